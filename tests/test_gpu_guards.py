"""GPU: the C entries of windows, drafted tokens and pages write nothing outside their tensors, whatever starts, lengths,
page numbers and the workspace's old contents are.  Outputs and workspaces lie between guards."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tests import seq_ref
from triton_fused_rope_flash_attn_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
PAD = 1 << 16
STARTS = [[0, 30, 10, 50, 40], [5, -9, 1 << 30, 7, 60], [60, 40, 20, 10, 0], [0, 200, 0, 200, 3], [0, 0, 130, 131, 200],
          [-(2 ** 31), 2 ** 31 - 1, -1, 190, 2 ** 31 - 1]]
OLD = [0, 0x7fffffff, -(2 ** 31), -1, 1]   # what a workspace held before, in 32-bit numbers; and random ones


class Guarded:
    """Bytes between two guards."""

    def __init__(self, nbytes, old=None, seed=0):
        self.n = nbytes
        self.buf = torch.full((2 * PAD + nbytes + 3,), 0xA5, dtype=torch.uint8, device=DEV)[: (2 * PAD + nbytes + 3) // 4 * 4]
        inner = self.buf[PAD:PAD + nbytes // 4 * 4].view(torch.int32)
        if old is None:
            inner.copy_(torch.randint(-2 ** 31, 2 ** 31 - 1, inner.shape, generator=torch.Generator().manual_seed(seed)).to(torch.int32))
        else:
            inner.fill_(old)
        self.ptr = self.buf.data_ptr() + PAD
        self.inner = inner

    def check(self):
        assert (self.buf[:PAD] == 0xA5).all() and (self.buf[PAD + self.n:] == 0xA5).all()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def randn(*shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def strides(t):
    return (ctypes.c_int64 * 3)(*t.stride()[-3:])


def desc(**kw):
    d = dict(tokens=0, seqs=4, heads=4, kv_heads=2, head_dim=64, n_pos=64, has_cls=1, causal=1, dtype=_lib.BF16, softmax_scale=0.125)
    d.update(kw)
    return _lib.SeqDesc(*d.values())


def cache_desc(kc, vc, pages):
    s = [(ctypes.c_int64 * 3)(*c.stride()[:3]) for c in (kc, vc)]
    return _lib.CacheDesc(kc.data_ptr(), vc.data_ptr(), *s, kc.shape[0], kc.shape[1], pages.shape[1], pages.stride(0))


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (F32, 32)])
@pytest.mark.parametrize("old", [*OLD, None])
def test_tree(dtype, D, old):
    lib, T, H, Hkv, page = _lib.load(), 200, 4, 2, 16
    es = 2 if dtype == BF16 else 4
    q, tree = randn(T, H, D, dtype=dtype, seed=1), torch.rand(T, 70, generator=torch.Generator().manual_seed(2)).to(DEV) < 0.5
    kc, vc = (randn(90, page, Hkv, D, dtype=dtype, seed=s) for s in (3, 4))
    want = kc.clone(), vc.clone()
    cos, sin = seq_ref.Table(64, D, DEV).tables()
    for per in (20, 60):                     # a workgroup a tile, and shares of all
        pages = torch.randint(-1, 92, (4, per), generator=torch.Generator().manual_seed(per)).to(torch.int32).to(DEV)
        c = cache_desc(kc, vc, pages)
        d = desc(tokens=T, head_dim=D, dtype=_lib.DTYPE_CODE[dtype])
        n = lib.farope_tree_workspace_elems(ctypes.byref(d), ctypes.byref(c))
        assert (n > 0) == (per * page > 512)
        for starts in STARTS:
            for lengths in ([9, 300, 4, 1], [-1, 2 ** 31 - 1, 0, 950]):
                for mask in (tree, None):
                    cu, at, o, ws = ints(starts), ints(lengths), Guarded(T * H * D * es), Guarded(4 * n, old)
                    rc = lib.farope_tree(ctypes.byref(d), q.data_ptr(), strides(q), cos.data_ptr(), sin.data_ptr(), None, ctypes.byref(c),
                                         pages.data_ptr(), at.data_ptr(), cu.data_ptr(), None if mask is None else mask.data_ptr(), 70, 70,
                                         o.ptr, ws.ptr, n, None)
                    assert rc == _lib.OK
                    torch.cuda.synchronize()
                    o.check()
                    ws.check()
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


@pytest.mark.parametrize("dtype,D,window,sinks", [(BF16, 64, 20, 4), (BF16, 128, 20, 70), (BF16, 128, 1, 0), (F32, 32, 9, 200), (BF16, 256, 30, 3)])
def test_window(dtype, D, window, sinks):
    lib, T, H, Hkv = _lib.load(), 200, 4, 2
    es = 2 if dtype == BF16 else 4
    q, do = (randn(T, H, D, dtype=dtype, seed=s) for s in (1, 2))
    k, v = (randn(T, Hkv, D, dtype=dtype, seed=s) for s in (3, 4))
    cos, sin = seq_ref.Table(64, D, DEV).tables()
    d = desc(tokens=T, head_dim=D, dtype=_lib.DTYPE_CODE[dtype])
    w = ctypes.byref(d), window, sinks
    qkv = (q.data_ptr(), strides(q), k.data_ptr(), strides(k), v.data_ptr(), strides(v))
    sizes = [lib.farope_seq_window_workspace_elems(*w, b, 1, 1) for b in (0, 1)]
    for i, starts in enumerate(STARTS):
        cu = ints(starts)
        o, lse, fws, bws = Guarded(T * H * D * es), Guarded(4 * T * H), *(Guarded(4 * n, None if i else 0x7f800000) for n in sizes)
        dq, dk, dv = (Guarded(T * h * D * es) for h in (H, Hkv, Hkv))
        tail = (cos.data_ptr(), sin.data_ptr(), None, cu.data_ptr())
        assert lib.farope_seq_window_fwd(*w, *qkv, *tail, o.ptr, lse.ptr, fws.ptr, sizes[0], None) == _lib.OK
        assert lib.farope_seq_window_bwd(*w, *qkv, o.ptr, do.data_ptr(), strides(do), lse.ptr, *tail, dq.ptr, dk.ptr, dv.ptr, bws.ptr,
                                         sizes[1], None) == _lib.OK
        torch.cuda.synchronize()
        for g in (o, lse, fws, bws, dq, dk, dv):
            g.check()


@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 5), (900, 1000), (2000, 3)])
def test_window_decode(window, sinks):
    lib, B, H, Hkv, D, page = _lib.load(), 4, 4, 2, 64, 16
    q = randn(B, H, D, dtype=BF16, seed=1)
    kc, vc = (randn(90, page, Hkv, D, dtype=BF16, seed=s) for s in (3, 4))
    cos, sin = seq_ref.Table(64, D, DEV).tables()
    for per in (20, 200):
        pages = torch.randint(-1, 92, (B, per), generator=torch.Generator().manual_seed(per)).to(torch.int32).to(DEV)
        c, d = cache_desc(kc, vc, pages), desc(tokens=B, head_dim=D)
        n = lib.farope_decode_window_workspace_elems(ctypes.byref(d), ctypes.byref(c), window, sinks)
        for old in (*OLD, None):
            for lengths in ([9, 300, 0, 1], [-1, 2 ** 31 - 1, -(2 ** 31), 3199]):
                at, o, ws = ints(lengths), Guarded(B * H * D * 2), Guarded(4 * n, old)
                rc = lib.farope_decode_window(ctypes.byref(d), window, sinks, q.data_ptr(), strides(q), cos.data_ptr(), sin.data_ptr(), None,
                                              ctypes.byref(c), pages.data_ptr(), at.data_ptr(), o.ptr, ws.ptr, n, None)
                assert rc == _lib.OK
                torch.cuda.synchronize()
                o.check()
                ws.check()


@pytest.mark.parametrize("seed", range(4))
def test_pages(seed):
    """Paths, parents, counts and tables of any values: only the cache's pages, the table, lengths and counts are written."""
    lib, B, Hkv, D, page, n_pages, per = _lib.load(), 40, 2, 64, 16, 1100, 30
    g = torch.Generator().manual_seed(seed)
    row = page * Hkv * D * 2
    s = (ctypes.c_int64 * 3)(page * Hkv * D, Hkv * D, D)

    def table(hi, shape):
        return torch.randint(-3, hi, shape, generator=g).to(torch.int32)

    def guarded(x):
        t = Guarded(4 * x.numel())
        t.inner.copy_(x.flatten())
        return t

    lengths = table(per * page + 50, (B,))
    lengths[:3] = torch.tensor([-(2 ** 31), 2 ** 31 - 1, per * page], dtype=torch.int32)
    kc, vc = Guarded(n_pages * row, 0), Guarded(n_pages * row, 0)
    c = _lib.CacheDesc(kc.ptr, vc.ptr, s, s, n_pages, page, per, per)
    d = desc(seqs=B, head_dim=D)
    pages, lens, out = guarded(table(n_pages + 3, (B, per))), guarded(lengths), Guarded(4 * B)
    path = table(40, (B, 33)) if seed % 2 else torch.randint(-2 ** 31, 2 ** 31 - 1, (B, 33), generator=g).abs().to(torch.int32)
    path = path.to(DEV)
    assert lib.farope_cache_accept(ctypes.byref(d), ctypes.byref(c), pages.ptr, lens.ptr, path.data_ptr(), 33, 33, out.ptr, None) == _lib.OK
    refs, missing = guarded(table(3, (n_pages,))), Guarded(4)
    parents, room = table(B + 3, (B,)).to(DEV), table(200, (B,))
    room[:2] = torch.tensor([2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32)
    room = room.to(DEV)
    n = lib.farope_cache_fork_workspace_elems(B, ctypes.byref(c))
    ws = Guarded(4 * n, [0x7fffffff, -1, 0, None][seed])
    assert lib.farope_cache_fork(ctypes.byref(d), ctypes.byref(c), pages.ptr, lens.ptr, refs.ptr, parents.data_ptr(), room.data_ptr(),
                                 missing.ptr, ws.ptr, n, None) == _lib.OK
    torch.cuda.synchronize()
    for t in (kc, vc, pages, lens, out, refs, missing, ws):
        t.check()
    assert ((lens.inner >= 0) & (lens.inner <= per * page)).all()
    assert ((pages.inner >= -1) & (pages.inner < n_pages)).all()
