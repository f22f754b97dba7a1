"""Refusals of windowed attention (the same cases on the GPU), its C entries' argument errors and workspaces."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tests import seq_ref
from tests.test_pages_cpu import DEVICES, _cache, _cdesc, _desc, _i
from triton_fused_rope_flash_attn_amd import _lib, sdpa_rope_decode, sdpa_rope_varlen


def _varlen(dev, **kw):
    q, k, v = (torch.zeros(10, h, 64, dtype=torch.bfloat16, device=dev) for h in (4, 2, 2))
    return sdpa_rope_varlen(q, k, v, seq_ref.Table(10, 64, dev), _i([0, 4, 10], dev), **kw)


def _decode(dev, **kw):
    return sdpa_rope_decode(torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=dev), cos_sin=seq_ref.Table(10, 64, dev), **_cache(dev), **kw)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("fn", [_varlen, _decode])
@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-1), dict(window=2 ** 31), dict(window=4, sinks=-1), dict(window=4, sinks=2 ** 31)])
def test_refuses(fn, kw, dev):
    with pytest.raises(ValueError, match="window must be at least 1"):
        fn(dev, **kw)


@pytest.mark.parametrize("dev", DEVICES)
def test_a_window_is_causal(dev):
    with pytest.raises(ValueError, match="causal"):
        _varlen(dev, window=4, causal=False)


@pytest.mark.parametrize("fn", [_varlen, _decode])
def test_cpu_tensors_are_refused(fn):
    with pytest.raises(RuntimeError, match="ROCm GPUs only"):
        fn("cpu", window=4)


def test_meta_tensors():
    q, k = (torch.empty(10, h, 64, dtype=torch.float16, device="meta") for h in (4, 2))
    c = torch.empty(5, 32, device="meta")
    cu = torch.empty(3, dtype=torch.int32, device="meta")
    o, lse = torch.ops.farope.seq_window_fwd(q, k, k, c, c, cu, None, True, 0.125, 4, 1)
    assert o.shape == q.shape and lse.shape == (4, 10) and lse.dtype == torch.float32
    grads = torch.ops.farope.seq_window_bwd(o, q, k, k, o, lse, c, c, cu, None, True, 0.125, 4, 1)
    assert [g.shape for g in grads] == [q.shape, k.shape, k.shape]


SHAPE, NULL = _lib.ERR_SHAPE, _lib.ERR_NULL


def test_c_entries_refuse():
    """(nothing is launched: every call has a mistake)"""
    lib, s = _lib.load(), (ctypes.c_int64 * 3)(256, 64, 1)
    d = _desc(tokens=1000, heads=4, n_pos=10)

    def fwd(window, sinks, d=d, q=16, n=1 << 40):
        return lib.farope_seq_window_fwd(ctypes.byref(d), window, sinks, q, s, 16, s, 16, s, 16, 16, None, 4, 16, 4, 16, n, None)

    def bwd(window, sinks, d=d, q=16, n=1 << 40):
        return lib.farope_seq_window_bwd(ctypes.byref(d), window, sinks, q, s, 16, s, 16, s, 16, 16, s, 4, 16, 16, None, 4, 16, 16, 16, 16, n, None)

    for fn in (fwd, bwd):
        assert fn(0, 0) == SHAPE and fn(-1, 0) == SHAPE and fn(4, -1) == SHAPE
        assert fn(4, 0, q=None) == NULL and fn(4, 0, n=1) == _lib.ERR_SCRATCH
        assert fn(4, 0, d=_desc(tokens=100, heads=3, n_pos=10)) == SHAPE
        assert fn(4, 0, d=_desc(tokens=0, heads=4, n_pos=10)) == _lib.OK
    assert lib.farope_seq_window_fwd(None, 1, 0, *[None] * 13, 0, None) == NULL

    one = _desc(tokens=2, heads=4, n_pos=10)

    def decode(window, sinks, q=16):
        return lib.farope_decode_window(ctypes.byref(one), window, sinks, q, s, 16, 16, None, ctypes.byref(_cdesc()), 64, 64, 16, 16, 0, None)

    assert decode(0, 0) == SHAPE and decode(4, -1) == SHAPE and decode(4, 0, q=None) == NULL
    assert lib.farope_decode_window(ctypes.byref(one), 1, 0, *[None] * 10, 0, None) == NULL


def test_c_workspaces():
    lib = _lib.load()

    def seq(window, sinks, backward=1, **kw):
        d = _desc(**{**dict(tokens=4096, seqs=1, heads=4, n_pos=10, dtype=_lib.BF16), **kw})
        args = (backward, 1, 1)
        return (lib.farope_seq_window_workspace_elems(ctypes.byref(d), window, sinks, *args),
                lib.farope_seq_workspace_elems(ctypes.byref(d), *args))

    assert seq(0, 0)[0] == 0 and seq(4, -1)[0] == 0
    for window in (4096, 1 << 30):   # a window that holds everything is none
        a, b = seq(window, 9)
        assert a == b
    a, b = seq(128, 0, 0)
    assert a == b                    # the forward's rows are the same
    none, _ = seq(128, 0)
    some, _ = seq(128, 65)
    # the sinks' tiles have 2 heads of 65 stages; other tiles 8, in 4 parts of 2: 65 parts of two tiles' sums, for K and V
    assert some - none == 2 * 65 * 2 * 64 * 2 * 64
    short, _ = seq(4000, 65)
    none, _ = seq(4000, 0)
    assert short == none             # the sinks' tiles have no more to do than others

    def decode(window, sinks, **kw):
        d = _desc(tokens=2, heads=4, n_pos=10, **kw)
        c = _cdesc(max_pages=1000)
        return (lib.farope_decode_window_workspace_elems(ctypes.byref(d), ctypes.byref(c), window, sinks),
                lib.farope_decode_workspace_elems(ctypes.byref(d), ctypes.byref(c)))

    assert decode(0, 0)[0] == 0 and decode(100, 4)[0] == 0 and decode(100, 4)[1] > 0   # (a worker a sequence)
    assert decode(16000, 0)[0] == decode(16000, 0)[1]
    assert 0 < decode(2000, 4)[0] < decode(16000, 0)[1]


# (the divided form of the sinks' tiles fits no launch, or is not taken: that is no reason to refuse)
@pytest.mark.parametrize("window,sinks,kw", [
    (128, 4096, dict(tokens=65536, seqs=256, heads=16, kv_heads=16)),
    (64, 4, dict(tokens=300000, seqs=40000, heads=8, kv_heads=8)),
    (64, 1024, dict(tokens=262144, seqs=4096, heads=8, kv_heads=8)),
    (512, 2 ** 31 - 1, dict(tokens=65536, seqs=16, heads=16, kv_heads=16)),
    (64, 4, dict(tokens=24000000, seqs=40000, heads=8, kv_heads=8, head_dim=32)),
    (2, 1, dict(tokens=16000000, seqs=260000, heads=1, kv_heads=1)),
])
def test_the_backward_takes_what_the_forward_takes(window, sinks, kw):
    """(nothing is launched: the forward's LSE is not aligned, the backward's workspace too short; both are looked at after the sizes)"""
    lib, s, d = _lib.load(), (ctypes.c_int64 * 3)(8, 8, 1), _desc(**{**dict(n_pos=10), **kw})
    fwd = lib.farope_seq_window_fwd(ctypes.byref(d), window, sinks, 16, s, 16, s, 16, s, 16, 16, None, 4, 16, 6, 16, 1, None)
    bwd = lib.farope_seq_window_bwd(ctypes.byref(d), window, sinks, 16, s, 16, s, 16, s, 16, 16, s, 4, 16, 16, None, 4, 16, 16, 16, 16, 1, None)
    assert (fwd, bwd) == (_lib.ERR_ALIGN, _lib.ERR_SCRATCH)


@pytest.mark.parametrize("dtype,D", [(_lib.BF16, 32), (_lib.F16, 64), (_lib.BF16, 128), (_lib.F16, 256), (_lib.F32, 64), (_lib.F32, 256)])
@pytest.mark.parametrize("tokens,seqs,heads,kv,window,sinks", [
    (16384, 1, 32, 8, 1024, 4), (16384, 1, 32, 8, 1024, 1024), (16384, 1, 32, 8, 1024, 4096), (131072, 32, 32, 8, 512, 2048),
    (16384, 8, 32, 8, 512, 1024), (131072, 8, 32, 8, 1024, 4), (65536, 64, 8, 8, 64, 4), (65536, 16, 16, 16, 512, 2 ** 31 - 1),
])
def test_many_sinks_need_no_more_workspace(dtype, D, tokens, seqs, heads, kv, window, sinks):
    """The sinks' sums are those of one resident round of workgroups at most, 2 * 64 * D each: 32 MB whatever the call."""
    lib = _lib.load()
    d = _desc(tokens=tokens, seqs=seqs, heads=heads, kv_heads=kv, head_dim=D, dtype=dtype, n_pos=10)
    with_, none = (lib.farope_seq_window_workspace_elems(ctypes.byref(d), window, s, 1, 1, 1) for s in (sinks, 0))
    assert 0 <= (with_ - none) * 4 <= 32 << 20
