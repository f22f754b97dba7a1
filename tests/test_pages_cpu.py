"""Refusals of the entry points that move rows and pages of a cache (the same cases on the GPU, where
the native kernels make the checks), and their C entries' argument errors."""
from __future__ import annotations

import ctypes

import pytest
import torch

from triton_fused_rope_flash_attn_amd import _lib, rope_cache_accept, rope_cache_fork

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _i(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _cache(dev):
    kc, vc = (torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16, device=dev) for _ in range(2))
    return dict(k_cache=kc, v_cache=vc, page_table=_i([[0, 1], [2, 3]], dev), lengths=_i([3, 17], dev))


def _accept_args(dev):
    return dict(**_cache(dev), path=_i([[0, 2], [1, -1]], dev))


def _fork_args(dev):
    return dict(**_cache(dev), refs=_i([1, 1, 1, 1, 0], dev), parents=_i([0, 0], dev), room=_i([1, 1], dev))


CACHE = [
    ("three dims", ValueError, lambda a: dict(k_cache=a["k_cache"][0])),
    ("caches differ", ValueError, lambda a: dict(v_cache=a["v_cache"][:4])),
    ("no pages", ValueError, lambda a: {n: a[n][:0] for n in ("k_cache", "v_cache")}),
    ("no rows", ValueError, lambda a: {n: a[n][:, :0] for n in ("k_cache", "v_cache")}),
    ("no heads", ValueError, lambda a: {n: a[n][:, :, :0] for n in ("k_cache", "v_cache")}),
    ("head_dim", ValueError, lambda a: {n: a[n][..., :48] for n in ("k_cache", "v_cache")}),
    ("dtype", TypeError, lambda a: {n: a[n].double() for n in ("k_cache", "v_cache")}),
    ("mixed dtypes", TypeError, lambda a: dict(v_cache=a["v_cache"].half())),
    ("channels apart", ValueError, lambda a: dict(k_cache=a["k_cache"].transpose(2, 3).contiguous().transpose(2, 3))),
    ("table's dtype", TypeError, lambda a: dict(page_table=a["page_table"].long())),
    ("table's shape", ValueError, lambda a: dict(page_table=a["page_table"][0])),
    ("table's columns apart", ValueError, lambda a: dict(page_table=a["page_table"].t())),
    ("lengths' dtype", TypeError, lambda a: dict(lengths=a["lengths"].long())),
    ("lengths' shape", ValueError, lambda a: dict(lengths=a["lengths"][:1])),
]
ACCEPT = CACHE + [
    ("path's dtype", TypeError, lambda a: dict(path=a["path"].long())),
    ("path's shape", ValueError, lambda a: dict(path=a["path"][0])),
    ("path's rows", ValueError, lambda a: dict(path=a["path"][:1])),
    ("path's columns apart", ValueError, lambda a: dict(path=a["path"].t())),
    ("path's width", ValueError, lambda a: dict(path=a["path"].new_zeros(2, 2049))),
]
FORK = CACHE + [
    ("table rows overlap", ValueError, lambda a: dict(page_table=a["page_table"][:1].expand(2, 2))),
    ("refs' dtype", TypeError, lambda a: dict(refs=a["refs"].long())),
    ("refs' shape", ValueError, lambda a: dict(refs=a["refs"][:4])),
    ("parents' dtype", TypeError, lambda a: dict(parents=a["parents"].long())),
    ("parents' shape", ValueError, lambda a: dict(parents=a["parents"][:1])),
    ("room's dtype", TypeError, lambda a: dict(room=a["room"].long())),
    ("room's shape", ValueError, lambda a: dict(room=a["room"][:1])),
]


def _refuses(fn, args, error, change):
    args.update(change(args))
    before = {n: t.clone() for n, t in args.items()}
    with pytest.raises(error):
        fn(**args)
    assert all(torch.equal(args[n], t) for n, t in before.items())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("what,error,change", ACCEPT, ids=[c[0] for c in ACCEPT])
def test_accept_refuses(what, error, change, dev):
    _refuses(rope_cache_accept, _accept_args(dev), error, change)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("what,error,change", FORK, ids=[c[0] for c in FORK])
def test_fork_refuses(what, error, change, dev):
    _refuses(rope_cache_fork, _fork_args(dev), error, change)


@pytest.mark.parametrize("fn,make", [(rope_cache_accept, _accept_args), (rope_cache_fork, _fork_args)])
def test_cpu_tensors_are_refused(fn, make):
    with pytest.raises(RuntimeError, match="ROCm GPUs only"):
        fn(**make("cpu"))


@pytest.mark.gpu
@pytest.mark.parametrize("fn,make", [(rope_cache_accept, _accept_args), (rope_cache_fork, _fork_args)])
def test_mixed_devices_are_refused(fn, make):
    for name in make("cpu"):
        if name != "k_cache":
            args = make("cuda")
            args[name] = args[name].cpu()
            with pytest.raises(RuntimeError, match="device"):
                fn(**args)


def _desc(**kw):
    d = dict(tokens=0, seqs=2, heads=2, kv_heads=2, head_dim=64, n_pos=0, has_cls=0, causal=0, dtype=_lib.BF16, softmax_scale=0.0)
    d.update(kw)
    return _lib.SeqDesc(*d.values())


def _cdesc(**kw):
    s = (ctypes.c_int64 * 3)(2048, 128, 64)
    d = dict(k=256, v=256, k_stride=s, v_stride=s, pages=5, page_rows=16, max_pages=2, table_stride=2)
    d.update(kw)
    return _lib.CacheDesc(*d.values())


NULL, ALIGN, SHAPE, SCRATCH = _lib.ERR_NULL, _lib.ERR_ALIGN, _lib.ERR_SHAPE, _lib.ERR_SCRATCH


def test_c_entries_refuse():
    """(nothing is launched: every call has a mistake)"""
    lib = _lib.load()

    def accept(d=None, c=None, table=64, lengths=64, path=64, stride=2, cols=2, out=64):
        return lib.farope_cache_accept(ctypes.byref(d or _desc()), ctypes.byref(c or _cdesc()), table, lengths, path, stride, cols, out, None)

    def fork(d=None, c=None, table=64, lengths=64, refs=64, parents=64, room=64, missing=64, ws=64, n=1 << 40):
        return lib.farope_cache_fork(ctypes.byref(d or _desc()), ctypes.byref(c or _cdesc()), table, lengths, refs, parents, room, missing,
                                     ws, n, None)

    for fn in (accept, fork):
        assert fn(_desc(seqs=0)) == SHAPE and fn(_desc(kv_heads=0)) == SHAPE and fn(_desc(head_dim=48)) == _lib.ERR_HEAD_DIM
        assert fn(_desc(dtype=7)) == _lib.ERR_DTYPE and fn(c=_cdesc(k=0)) == NULL and fn(c=_cdesc(v=8)) == ALIGN
        assert fn(c=_cdesc(pages=0)) == SHAPE and fn(c=_cdesc(page_rows=0)) == SHAPE and fn(c=_cdesc(max_pages=0)) == SHAPE
        assert fn(c=_cdesc(k_stride=(ctypes.c_int64 * 3)(2048, 128, 60))) == ALIGN
        assert fn(table=None) == NULL and fn(lengths=2) == ALIGN
        assert fn(_desc(seqs=1 << 24)) == SHAPE
    assert accept(path=None) == NULL and accept(cols=-1) == SHAPE and accept(cols=2049) == SHAPE and accept(stride=-1) == SHAPE
    assert accept(out=None) == NULL
    assert fork(refs=None) == NULL and fork(parents=None) == NULL and fork(room=2) == ALIGN and fork(missing=None) == NULL
    assert fork(ws=None) == NULL and fork(n=10) == SCRATCH and fork(c=_cdesc(table_stride=1)) == SHAPE
    assert lib.farope_cache_accept(None, None, None, None, None, 0, 0, None, None) == NULL
    assert lib.farope_cache_fork(None, None, None, None, None, None, None, None, None, 0, None) == NULL


def test_c_fork_workspace():
    lib = _lib.load()
    assert lib.farope_cache_fork_workspace_elems(0, ctypes.byref(_cdesc())) == 0
    assert lib.farope_cache_fork_workspace_elems(2, None) == 0
    # bits of 1024 pages, a count, the table, three numbers a place, the pages given out; parts of 4
    assert lib.farope_cache_fork_workspace_elems(2, ctypes.byref(_cdesc())) == 32 + 4 + 4 + 3 * 4 + 4
    assert lib.farope_cache_fork_workspace_elems(3, ctypes.byref(_cdesc(pages=2000, max_pages=7))) == 64 + 4 + 24 + 12 + 24
