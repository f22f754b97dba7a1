"""Refusals of the packed and cached attention's entry points (the same cases on the
GPU, where the native kernels make the checks), their C entries' argument errors, and
the reference's gradients."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tests import seq_ref
from triton_fused_rope_flash_attn_amd import _lib, rope_cache_append, sdpa_rope_decode, sdpa_rope_varlen

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _i(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _varlen_args(dev, D=64, dtype=torch.bfloat16):
    q, k, v = (torch.zeros(10, h, D, dtype=dtype, device=dev) for h in (4, 2, 2))
    return dict(Q=q, K=k, V=v, cos_sin=seq_ref.Table(10, 64, dev), cu_seqlens=_i([0, 4, 10], dev))


def _cache_args(dev, dtype=torch.bfloat16):
    kc, vc = (torch.zeros(5, 16, 2, 64, dtype=dtype, device=dev) for _ in range(2))
    return dict(cos_sin=seq_ref.Table(10, 64, dev), k_cache=kc, v_cache=vc, page_table=_i([[0, 1], [2, 3]], dev),
                lengths=_i([3, 17], dev))


def _append_args(dev):
    k, v = (torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=dev) for _ in range(2))
    return dict(K=k, V=v, **_cache_args(dev))


def _decode_args(dev):
    return dict(Q=torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=dev), **_cache_args(dev))


class _Tables:
    def __init__(self, c, s):
        self.c, self.s = c, s

    def tables(self):
        return self.c, self.s


VARLEN = [
    ("two dims", ValueError, lambda a: dict(Q=a["Q"][0])),
    ("K and V differ", ValueError, lambda a: dict(V=a["V"][:, :1])),
    ("tokens differ", ValueError, lambda a: dict(K=a["K"][:9], V=a["V"][:9])),
    ("heads not a multiple", ValueError, lambda a: dict(Q=a["Q"][:, :3])),
    ("no heads", ValueError, lambda a: dict(Q=a["Q"][:, :0])),
    ("head_dim", ValueError, lambda a: {n: a[n][..., :48] for n in "QKV"}),
    ("no channels", ValueError, lambda a: {n: a[n][..., :0] for n in "QKV"}),
    ("dtype", TypeError, lambda a: {n: a[n].double() for n in "QKV"}),
    ("mixed dtypes", TypeError, lambda a: dict(K=a["K"].half())),
    ("starts' dtype", TypeError, lambda a: dict(cu_seqlens=a["cu_seqlens"].long())),
    ("starts' shape", ValueError, lambda a: dict(cu_seqlens=a["cu_seqlens"][None])),
    ("starts apart", ValueError, lambda a: dict(cu_seqlens=torch.stack([a["cu_seqlens"]] * 2, 1)[:, 0])),
    ("no sequence", ValueError, lambda a: dict(cu_seqlens=a["cu_seqlens"][:1])),
    ("positions' dtype", TypeError, lambda a: dict(positions=torch.zeros(10, device=a["Q"].device))),
    ("positions' length", ValueError, lambda a: dict(positions=_i([0] * 9, a["Q"].device))),
    ("table's width", ValueError, lambda a: dict(cos_sin=seq_ref.Table(10, 128, a["Q"].device))),
    ("table's dtype", ValueError, lambda a: dict(cos_sin=_Tables(*(t.double() for t in a["cos_sin"].tables())))),
    ("tables differ", ValueError, lambda a: dict(cos_sin=_Tables(a["cos_sin"].cos, a["cos_sin"].sin[:5]))),
    ("no table rows", ValueError, lambda a: dict(cos_sin=_Tables(*(t[:0] for t in a["cos_sin"].tables())))),
]
CACHE = [
    ("cache dims", ValueError, lambda a: dict(k_cache=a["k_cache"][0])),
    ("cache heads", ValueError, lambda a: dict(k_cache=a["k_cache"][:, :, :0], v_cache=a["v_cache"][:, :, :0])),
    ("caches differ", ValueError, lambda a: dict(v_cache=a["v_cache"][:4])),
    ("no pages", ValueError, lambda a: dict(k_cache=a["k_cache"][:0], v_cache=a["v_cache"][:0])),
    ("cache dtype", TypeError, lambda a: dict(k_cache=a["k_cache"].half())),
    ("cache channels apart", ValueError, lambda a: dict(k_cache=torch.stack([a["k_cache"]] * 2, -1)[..., 0])),
    ("cache rows not aligned", ValueError,
     lambda a: dict(k_cache=torch.zeros(5, 16, 2, 65, dtype=torch.bfloat16, device=a["lengths"].device)[..., :64])),
    ("page table's dtype", TypeError, lambda a: dict(page_table=a["page_table"].long())),
    ("page table's dims", ValueError, lambda a: dict(page_table=a["page_table"][0])),
    ("page table's rows apart", ValueError, lambda a: dict(page_table=a["page_table"].t())),
    ("no page entries", ValueError, lambda a: dict(page_table=a["page_table"][:, :0])),
    ("lengths' dtype", TypeError, lambda a: dict(lengths=a["lengths"].long())),
    ("lengths' number", ValueError, lambda a: dict(lengths=a["lengths"][:1])),
    ("table's width", ValueError, lambda a: dict(cos_sin=seq_ref.Table(10, 32, a["lengths"].device))),
    ("positions' length", ValueError, lambda a: dict(positions=_i([0], a["lengths"].device))),
]
APPEND = CACHE + [
    ("two dims", ValueError, lambda a: dict(K=a["K"][0], V=a["V"][0])),
    ("K and V differ", ValueError, lambda a: dict(V=a["V"][:, :1])),
    ("mixed dtypes", TypeError, lambda a: dict(V=a["V"].half())),
    ("tokens and sequences", ValueError, lambda a: dict(K=a["K"][:1], V=a["V"][:1])),
    ("starts and sequences", ValueError, lambda a: dict(cu_seqlens=_i([0, 2], a["K"].device))),
]
DECODE = CACHE + [
    ("two dims", ValueError, lambda a: dict(Q=a["Q"][0])),
    ("heads not a multiple", ValueError, lambda a: dict(Q=a["Q"][:, :3])),
    ("queries and sequences", ValueError, lambda a: dict(Q=a["Q"][:1])),
    ("query dtype", TypeError, lambda a: dict(Q=a["Q"].float())),
]


def _refused(fn, make, what, error, change, dev):
    args = make(dev)
    args.update(change(args))
    with pytest.raises(error):
        fn(**args)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("what,error,change", VARLEN, ids=[c[0] for c in VARLEN])
def test_varlen_refuses(what, error, change, dev):
    _refused(sdpa_rope_varlen, _varlen_args, what, error, change, dev)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("what,error,change", APPEND, ids=[c[0] for c in APPEND])
def test_append_refuses(what, error, change, dev):
    _refused(rope_cache_append, _append_args, what, error, change, dev)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("what,error,change", DECODE, ids=[c[0] for c in DECODE])
def test_decode_refuses(what, error, change, dev):
    _refused(sdpa_rope_decode, _decode_args, what, error, change, dev)


@pytest.mark.parametrize("fn,make", [(sdpa_rope_varlen, _varlen_args), (rope_cache_append, _append_args),
                                     (sdpa_rope_decode, _decode_args)])
def test_cpu_tensors_are_refused(fn, make):
    with pytest.raises(RuntimeError, match="ROCm GPUs only"):
        fn(**make("cpu"))


@pytest.mark.gpu
@pytest.mark.parametrize("fn,make,name", [(sdpa_rope_varlen, _varlen_args, "cu_seqlens"), (rope_cache_append, _append_args, "lengths"),
                                          (sdpa_rope_decode, _decode_args, "page_table"), (sdpa_rope_decode, _decode_args, "cos_sin")])
def test_mixed_devices_are_refused(fn, make, name):
    args = make("cuda")
    args[name] = make("cpu")[name]
    with pytest.raises(RuntimeError):
        fn(**args)


# ---------------------------------------------------------------------------
# the C entries: argument errors come before any launch
# ---------------------------------------------------------------------------
S3 = _lib.Stride3(128, 64, 1)


def _seq_desc(**kw):
    a = dict(tokens=10, seqs=2, heads=4, kv_heads=2, head_dim=64, n_pos=10, has_cls=1, causal=1, dtype=_lib.BF16)
    a.update(kw)
    return _lib.SeqDesc(*a.values(), 0.125)


def _fwd(desc, q=16, cu=16, o=16, ws=16, elems=1 << 20, cos=16):
    return _lib.load().farope_seq_fwd(ctypes.byref(desc), q, S3, 16, S3, 16, S3, cos, 16, None, cu, o, 16, ws, elems, None)


def _cache_desc(**kw):
    c = _lib.CacheDesc(16, 16, (2048, 128, 64), (2048, 128, 64), 5, 16, 2, 2)
    for n, x in kw.items():
        setattr(c, n, x)
    return c


@pytest.mark.parametrize("kw,rc", [
    (dict(seqs=0), _lib.ERR_SHAPE), (dict(tokens=-1), _lib.ERR_SHAPE), (dict(heads=3), _lib.ERR_SHAPE),
    (dict(kv_heads=0), _lib.ERR_SHAPE), (dict(head_dim=48), _lib.ERR_HEAD_DIM), (dict(dtype=5), _lib.ERR_DTYPE),
    (dict(n_pos=0), _lib.ERR_TABLE), (dict(has_cls=2), _lib.ERR_SEQ_LEN),
    (dict(tokens=1 << 25), _lib.ERR_SHAPE),                              # workspace rows past 32-bit offsets
    (dict(heads=1 << 18, kv_heads=1 << 18), _lib.ERR_SHAPE),             # output rows too wide
    (dict(seqs=1 << 23), _lib.ERR_SHAPE),                                # more slots than a launch holds
])
def test_c_entries_refuse_descriptors(kw, rc):
    desc = _seq_desc(**kw)
    assert _fwd(desc) == rc
    assert _lib.load().farope_seq_bwd(ctypes.byref(desc), 16, S3, 16, S3, 16, S3, 16, 16, S3, 16, 16, 16, None, 16, 16, 16, 16, 16,
                                      1 << 20, None) == rc


def _map_elems(tokens, seqs):
    """The tiles' places: 4 integers for each of (T >> 6) + B + 1 slots, in parts of 64."""
    return -(-4 * ((tokens >> 6) + seqs + 1) // 64) * 64


def test_c_entries_refuse_pointers_and_workspaces():
    lib, d = _lib.load(), _seq_desc(tokens=1000)
    assert _fwd(d, q=None) == _lib.ERR_NULL and _fwd(d, cu=None) == _lib.ERR_NULL and _fwd(d, ws=None) == _lib.ERR_NULL
    assert _fwd(d, q=17) == _lib.ERR_ALIGN and _fwd(d, o=24) == _lib.ERR_ALIGN and _fwd(d, cos=20) == _lib.ERR_ALIGN
    n = lib.farope_seq_workspace_elems(ctypes.byref(d), 0, 1, 1)
    assert n > 0 and _fwd(d, elems=n - 1) == _lib.ERR_SCRATCH
    short = _seq_desc()                                  # short sequences: K is rotated by the tiles
    assert lib.farope_seq_workspace_elems(ctypes.byref(short), 0, 1, 1) == 0
    assert lib.farope_seq_workspace_elems(ctypes.byref(short), 0, 0, 1) == 2 * 10 * 2 * 64 // 2 + _map_elems(10, 2)
    assert lib.farope_seq_workspace_elems(ctypes.byref(_seq_desc(head_dim=48)), 0, 1, 1) == 0
    assert _fwd(_seq_desc(tokens=0)) == _lib.OK   # nothing to do
    assert lib.farope_seq_fwd(None, 16, S3, 16, S3, 16, S3, 16, 16, None, 16, 16, 16, 16, 0, None) == _lib.ERR_NULL


def test_c_workspace_parts():
    """K-hat and the tiles' places (the backward: of queries and of keys); a copy of V and of dO where their rows cannot be streamed; Q-hat and two row values;
    where key tiles are few, the parts' sums of dK and dV."""
    lib = _lib.load()
    d = _seq_desc(tokens=8000, heads=20, kv_heads=10, head_dim=128)
    kv, q, row = 8000 * 10 * 128 // 2, 8000 * 20 * 128 // 2, 8000 * 20
    size = lambda d, *a: lib.farope_seq_workspace_elems(ctypes.byref(d), *a)  # noqa: E731
    m = _map_elems(8000, 2)
    assert size(d, 0, 1, 1) == kv + m and size(d, 0, 0, 1) == 2 * kv + m
    assert size(d, 1, 1, 1) == kv + 2 * m + q + 2 * row and size(d, 1, 0, 0) == 2 * kv + 2 * m + 2 * q + 2 * row
    d = _seq_desc(tokens=4096, seqs=1, heads=4, kv_heads=4, head_dim=128)   # 4 x 66 workgroups: 4 parts
    n = 4096 * 4 * 128
    m = _map_elems(4096, 1)
    assert size(d, 0, 1, 1) == n // 2 + m and size(d, 1, 1, 1) == n + 2 * m + 2 * 4096 * 4 + 2 * 4 * n


@pytest.mark.parametrize("stride,ptr,ok", [
    ((128, 64, 1), 16, 1), ((0, 64, 1), 16, 1), ((64, 640, 1), 16, 1),
    ((128, 64, 2), 16, 0), ((128, 64, 1), 18, 0), ((129, 64, 1), 16, 0), ((128, 65, 1), 16, 0), ((-128, 64, 1), 16, 0),
    ((1 << 27, 64, 1), 16, 0),                                            # rows past 2 GiB
])
def test_c_streams(stride, ptr, ok):
    assert _lib.load().farope_seq_streams(ctypes.byref(_seq_desc()), ptr, _lib.Stride3(*stride)) == ok


def test_c_cache_entries_refuse():
    lib = _lib.load()

    def append(d, c, cu=None, lengths=16):
        return lib.farope_cache_append(ctypes.byref(d), 16, S3, 16, S3, 16, 16, None, ctypes.byref(c), 16, lengths, cu, None)

    def decode(d, c, ws=16, elems=1 << 24):
        return lib.farope_decode(ctypes.byref(d), 16, S3, 16, 16, None, ctypes.byref(c), 16, 16, 16, ws, elems, None)

    one = _seq_desc(tokens=2)
    assert append(_seq_desc(), _cache_desc()) == _lib.ERR_SHAPE          # 10 tokens of 2 sequences, no starts
    assert append(one, _cache_desc(), lengths=None) == _lib.ERR_NULL
    assert decode(_seq_desc(), _cache_desc()) == _lib.ERR_SHAPE
    for bad, rc in ((dict(pages=0), _lib.ERR_SHAPE), (dict(page_rows=0), _lib.ERR_SHAPE), (dict(max_pages=0), _lib.ERR_SHAPE),
                    (dict(k=None), _lib.ERR_NULL), (dict(v=24), _lib.ERR_ALIGN),
                    (dict(k_stride=(ctypes.c_int64 * 3)(2048, 127, 64)), _lib.ERR_ALIGN)):
        assert append(one, _cache_desc(**bad)) == rc and decode(one, _cache_desc(**bad)) == rc, bad
    long = _cache_desc(max_pages=1000)
    n = lib.farope_decode_workspace_elems(ctypes.byref(one), ctypes.byref(long))
    assert n > 0 and decode(one, long, elems=n - 1) == _lib.ERR_SCRATCH and decode(one, long, ws=None) == _lib.ERR_NULL


@pytest.mark.parametrize("D,dtype,most", [(128, _lib.BF16, 512), (256, _lib.F16, 256), (64, _lib.BF16, 768), (32, _lib.F16, 1024),
                                          (128, _lib.F32, 256)])
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (3, 1), (4, 4), (5, 1), (6, 2), (7, 1), (11, 3), (12, 1), (3, 20), (600, 1)])
def test_decode_workers_are_resident_at_once(kv_heads, group, D, dtype, most):
    """Equal shares of the cached rows: one round of workgroups, no few of them behind it."""
    heads, seqs, tiles = kv_heads * group, 4, -(-group // 16)
    d = _seq_desc(tokens=seqs, seqs=seqs, heads=heads, kv_heads=kv_heads, head_dim=D, dtype=dtype)
    n = _lib.load().farope_decode_workspace_elems(ctypes.byref(d), ctypes.byref(_cache_desc(max_pages=1 << 16)))
    # sums [workers + seqs, heads, D], two statistics each, rounded up to 4; owners [seqs, 2]
    workers = (n - 2 * seqs) // (heads * (D + 2)) - seqs
    assert (workers + seqs) * heads * (D + 2) <= n - 2 * seqs < (workers + seqs) * heads * (D + 2) + 4
    assert workers == max(1, most // (kv_heads * tiles))


def test_slots_cover_every_tile():
    """The grid's rule: sequence i takes slots (cu[i] >> lb) + i on, at least as many as it has tiles."""
    g = torch.Generator().manual_seed(0)
    for lb in (4, 6, 7):
        for _ in range(200):
            B = int(torch.randint(1, 9, (1,), generator=g))
            lens = [int(x) for x in torch.randint(0, 3 << lb, (B,), generator=g)]
            tail = int(torch.randint(0, 200, (1,), generator=g))
            cu = [sum(lens[:i]) for i in range(B + 1)]
            T = cu[-1] + tail
            first = [(c >> lb) + i for i, c in enumerate(cu)] + [(T >> lb) + B + 1]
            for i, n in enumerate([*lens, tail]):
                assert first[i + 1] - first[i] >= -(-n >> lb) if n else True
            assert first[-1] == (T >> lb) + B + 1


def test_reference_gradients_are_the_forwards():
    """The 64-bit reference's gradients against autograd of its forward's formula."""
    D, lens = 32, [5, 0, 9]
    T, cu = sum(lens), [0, 5, 5, 14]
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(T, h, D, generator=g, dtype=torch.float64, requires_grad=True) for h in (4, 2, 2))
    do = torch.randn(T, 4, D, generator=g, dtype=torch.float64)
    table = seq_ref.Table(9, D)
    ref = seq_ref.varlen(q, k, v, do, table, cu, True, True)
    total = 0.0
    for a, b in zip(cu[:-1], cu[1:]):
        if a == b:
            continue
        index = torch.arange(b - a) - 1
        qh, kh = seq_ref.rotate(q[a:b], table, index), seq_ref.rotate(k[a:b], table, index)
        s = torch.einsum("ihd,jhd->hij", qh, kh.repeat_interleave(2, 1)) / D ** 0.5
        s = s.masked_fill(torch.ones(b - a, b - a).triu(1).bool(), float("-inf"))
        o = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v[a:b].repeat_interleave(2, 1))
        assert torch.allclose(o, ref["o"][a:b])
        total = total + (o * do[a:b]).sum()
    for x, n in zip(torch.autograd.grad(total, (q, k, v)), ("dq", "dk", "dv")):
        assert torch.allclose(x, ref[n]), n
