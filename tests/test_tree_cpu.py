"""Refusals of attention of several new tokens over a cache (the same cases on the GPU, where the
native kernel makes the checks), and its C entry's argument errors."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tests import seq_ref
from tests.test_pages_cpu import CACHE, DEVICES, _cache, _cdesc, _desc, _i
from triton_fused_rope_flash_attn_amd import _lib, sdpa_rope_tree


def _args(dev):
    return dict(Q=torch.zeros(5, 4, 64, dtype=torch.bfloat16, device=dev), cos_sin=seq_ref.Table(10, 64, dev), **_cache(dev),
                cu_seqlens=_i([0, 2, 5], dev), tree=torch.ones(5, 3, dtype=torch.bool, device=dev), positions=_i([0] * 5, dev))


TREE = [c for c in CACHE if c[0] not in ("head_dim", "dtype")] + [
    ("two dims", ValueError, lambda a: dict(Q=a["Q"][0])),
    ("heads not a multiple", ValueError, lambda a: dict(Q=a["Q"][:, :3])),
    ("no query heads", ValueError, lambda a: dict(Q=a["Q"][:, :0])),
    ("head_dim", ValueError, lambda a: dict(Q=a["Q"][..., :48])),
    ("another head_dim", ValueError, lambda a: dict(Q=a["Q"][..., :32], cos_sin=seq_ref.Table(10, 32, a["Q"].device))),
    ("dtype", TypeError, lambda a: dict(Q=a["Q"].double())),
    ("another dtype", TypeError, lambda a: dict(Q=a["Q"].half())),
    ("tables", ValueError, lambda a: dict(cos_sin=seq_ref.Table(10, 32, a["Q"].device))),
    ("starts' dtype", TypeError, lambda a: dict(cu_seqlens=a["cu_seqlens"].long())),
    ("starts' number", ValueError, lambda a: dict(cu_seqlens=a["cu_seqlens"][:2])),
    ("tree's dtype", TypeError, lambda a: dict(tree=a["tree"].to(torch.uint8))),
    ("tree's shape", ValueError, lambda a: dict(tree=a["tree"][0])),
    ("tree's rows", ValueError, lambda a: dict(tree=a["tree"][:4])),
    ("tree's columns apart", ValueError, lambda a: dict(tree=a["tree"].new_ones(3, 5).t())),
    ("positions' dtype", TypeError, lambda a: dict(positions=a["positions"].long())),
    ("positions' number", ValueError, lambda a: dict(positions=a["positions"][:4])),
]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("what,error,change", TREE, ids=[c[0] for c in TREE])
def test_tree_refuses(what, error, change, dev):
    args = _args(dev)
    args.update(change(args))
    with pytest.raises(error):
        sdpa_rope_tree(**args)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="ROCm GPUs only"):
        sdpa_rope_tree(**_args("cpu"))


@pytest.mark.gpu
def test_mixed_devices_are_refused():
    for name in ("k_cache", "v_cache", "page_table", "lengths", "cu_seqlens", "tree", "positions"):
        args = _args("cuda")
        args[name] = args[name].cpu()
        with pytest.raises(RuntimeError, match="device"):
            sdpa_rope_tree(**args)


NULL, ALIGN, SHAPE, SCRATCH = _lib.ERR_NULL, _lib.ERR_ALIGN, _lib.ERR_SHAPE, _lib.ERR_SCRATCH


def test_c_entry_refuses():
    """(nothing is launched: every call has a mistake)"""
    lib, strides = _lib.load(), (ctypes.c_int64 * 3)(256, 64, 1)

    def call(d=None, c=None, q=16, s=strides, cos=16, sin=16, pos=None, table=64, lengths=64, cu=64, tree=1, stride=3, cols=3, o=16, ws=16,
             n=1 << 40):
        d = d or _desc(tokens=5, heads=4, n_pos=10)
        return lib.farope_tree(ctypes.byref(d), q, s, cos, sin, pos, ctypes.byref(c or _cdesc()), table, lengths, cu, tree, stride, cols, o,
                               ws, n, None)

    assert call(_desc(tokens=0, heads=4, n_pos=10)) == _lib.OK
    assert call(_desc(tokens=5, heads=3, n_pos=10)) == SHAPE and call(_desc(tokens=-1, heads=4, n_pos=10)) == SHAPE
    assert call(_desc(tokens=5, heads=4)) == _lib.ERR_TABLE and call(_desc(tokens=5, heads=4, n_pos=10, head_dim=48)) == _lib.ERR_HEAD_DIM
    assert call(q=None) == NULL and call(q=1) == ALIGN and call(s=None) == NULL and call(cos=4) == ALIGN and call(sin=None) == NULL
    assert call(pos=2) == ALIGN and call(table=None) == NULL and call(lengths=2) == ALIGN and call(cu=None) == NULL
    assert call(c=_cdesc(k=0)) == NULL and call(c=_cdesc(pages=0)) == SHAPE
    assert call(stride=-1) == SHAPE and call(cols=-1) == SHAPE and call(o=8) == ALIGN
    wide = _cdesc(max_pages=1000, table_stride=1000)
    assert call(c=wide, ws=None) == NULL and call(c=wide, n=100) == SCRATCH
    assert call(_desc(tokens=1 << 30, heads=4, n_pos=10)) == SHAPE and call(_desc(tokens=1 << 25, heads=64, kv_heads=64, n_pos=10)) == SHAPE
    assert lib.farope_tree(None, *[None] * 9, None, 0, 0, None, None, 0, None) == NULL


def test_c_workspace():
    lib = _lib.load()

    def elems(c, **kw):
        return lib.farope_tree_workspace_elems(ctypes.byref(_desc(**{**dict(tokens=5, heads=4, n_pos=10), **kw})), ctypes.byref(c))

    assert elems(_cdesc()) == 0                                             # a workgroup a tile
    assert elems(_cdesc(max_pages=100), heads=3) == 0 and elems(_cdesc(max_pages=0)) == 0
    # 3 places for tiles of 25 stages (1600 rows), 2 stages a worker at least: 39 workers; two pieces of 64 rows of each
    # worker and key head, their statistics, 4 integers a place
    rows = 2 * 39 * 2 * 64
    assert elems(_cdesc(max_pages=100)) == rows * 64 + 2 * rows + 4 * 3
    # more rows than a tile of 64 (16 bits): tiles of 128
    rows = 2 * 256 * 2 * 128
    assert elems(_cdesc(max_pages=10000), tokens=100) == rows * 64 + 2 * rows + 4 * 4
    assert elems(_cdesc(max_pages=10000), tokens=100, dtype=_lib.F32) == rows // 2 * 64 + rows + 4 * 6
