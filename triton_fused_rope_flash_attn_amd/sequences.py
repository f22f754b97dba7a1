"""Rotary attention of sequence models: packed sequences and a paged cache.

Next to the dense planes of ``attention.py``, for models that read or write
their tokens in order (an autoregressive generator over a token grid, a text
decoder), with the same tables, rotation and class-token convention:

* ``sdpa_rope_varlen``   attention over packed sequences of different lengths,
                         causal or not, with shared key heads; forward and gradients;
* ``rope_cache_append``  new keys (rotated on the way) and values into a paged cache;
* ``sdpa_rope_decode``   one new token per sequence over its cached keys;
* ``sdpa_rope_tree``     several new tokens per sequence over them: a drafted tree, or a chunk of a prompt.

The reference has no counterpart: its calls are dense [B, H, N, D] planes.

Tables are ``CosSinTable`` or any object whose ``tables()`` gives fp32 cosines
and sines ``[rows, D/2]``, channel pairs (2p, 2p+1), so one-dimensional positions
are a table of their own.  Token i of a sequence takes row ``i - has_cls`` (the
class token, i = 0 with ``has_cls``, is not rotated), or ``positions[t]``; a row
below 0 is not rotated, and one past the table takes its last row.

Sequence starts, lengths and page numbers stay on the GPU: no call waits for
the device, and a captured call reads their new values when it is replayed.
Their values are therefore not refused; each function says what it does with
those that make no sense, and none reads or writes outside its tensors.

The work is done by ``torch.library`` ops with native GPU kernels
(csrc/torch_seq_ops.cpp), one call into libfarope.so each, on the current stream of
the tensors' device.  There is no CPU fallback: CPU tensors raise.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .attention import _check_device, _sdpa_comp_dtype

__all__ = ["sdpa_rope_varlen", "rope_cache_append", "sdpa_rope_decode", "sdpa_rope_tree"]

HEAD_DIMS = (32, 64, 128, 256)


# ---------------------------------------------------------------------------
# argument checks of the ops' Python bodies (CPU and meta tensors); the native
# kernels make the same ones, with the same exceptions
# ---------------------------------------------------------------------------
def _check_first(x, name, shape):
    if x.dim() != 3:
        raise ValueError(f"{name} must be {shape}; got shape {tuple(x.shape)}")
    if x.shape[2] not in HEAD_DIMS:
        raise ValueError(f"farope: head_dim must be 32, 64, 128 or 256; got {x.shape[2]}")
    if x.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"farope: unsupported tensor dtype {x.dtype}")


def _check_like(x, name, q):
    if x.dtype != q.dtype:
        raise TypeError(f"farope: {name} must share the other tensors' dtype; got {x.dtype} and {q.dtype}")
    if x.device != q.device:
        raise RuntimeError(f"farope: {name} must be on the other tensors' device")


def _check_kv(k, v):
    if k.shape != v.shape or k.dim() != 3 or k.shape[1] < 1:
        raise ValueError(f"K and V must have the same shape; got {tuple(k.shape)} and {tuple(v.shape)}")


def _check_ints(x, name, n, q):
    if x.dtype != torch.int32:
        raise TypeError(f"farope: {name} must be int32; got {x.dtype}")
    if x.dim() != 1 or (n is not None and x.shape[0] != n) or not x.is_contiguous():
        raise ValueError(f"farope: {name} must be contiguous with {'one dimension' if n is None else f'{n} elements'}; "
                         f"got shape {tuple(x.shape)}")
    if x.device != q.device:
        raise RuntimeError(f"farope: {name} must be on the other tensors' device")


def _check_cu(cu, q):
    _check_ints(cu, "cu_seqlens", None, q)
    if cu.shape[0] < 2:
        raise ValueError("farope: cu_seqlens must hold at least one sequence (2 elements)")


def _check_tables(cosp, sinp, q):
    want = q.shape[2] // 2
    for t in (cosp, sinp):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape[0] < 1 or t.shape[1] != want or not t.is_contiguous():
            raise ValueError(f"farope: RoPE tables must be contiguous fp32 [n_pos, {want}]; got {t.dtype} {tuple(t.shape)}")
        if t.device != q.device:
            raise RuntimeError(f"farope: RoPE tables on {t.device}, tensors on {q.device}")
    if cosp.shape != sinp.shape:
        raise ValueError(f"farope: RoPE tables must be contiguous fp32 [n_pos, {want}]; got {tuple(cosp.shape)} and {tuple(sinp.shape)}")


def _check_cache(k_cache, v_cache, page_table, lengths, kv_heads, x):
    want = (kv_heads, x.shape[2])
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or tuple(k_cache.shape[2:]) != want:
        raise ValueError(f"farope: the caches must be [pages, page_rows, Hkv, D] with Hkv={want[0]}, D={want[1]}; "
                         f"got {tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    if k_cache.shape[0] < 1 or k_cache.shape[1] < 1:
        raise ValueError(f"farope: the caches have no rows: {tuple(k_cache.shape)}")
    for t, name in ((k_cache, "the key cache"), (v_cache, "the value cache")):
        _check_like(t, name, x)
        if t.stride(3) != 1 or any(s * t.element_size() % 16 for s in t.stride()[:3]):
            raise ValueError("farope: cache rows must have contiguous channels and be 16-byte aligned")
    if page_table.dtype != torch.int32:
        raise TypeError(f"farope: page_table must be int32; got {page_table.dtype}")
    if page_table.dim() != 2 or page_table.shape[1] < 1 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError(f"farope: page_table must be [B, max_pages], its rows contiguous; got shape {tuple(page_table.shape)}")
    if page_table.device != x.device:
        raise RuntimeError("farope: page_table must be on the other tensors' device")
    _check_ints(lengths, "lengths", page_table.shape[0], x)


def _check_window(window, sinks):
    if not (1 <= window < 2 ** 31 and 0 <= sinks < 2 ** 31):
        raise ValueError(f"farope: window must be at least 1 and sinks at least 0, both in 32 bits; got {window} and {sinks}")


def _check_seq(q, k, v, cosp, sinp, cu, positions):
    if q.dim() != 3:
        raise ValueError(f"Q must be [T, H, D]; got shape {tuple(q.shape)}")
    _check_kv(k, v)
    if k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError(f"Q and K must agree in tokens and head_dim; got {tuple(q.shape)} and {tuple(k.shape)}")
    if q.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError(f"farope: query heads must be a multiple of key heads; got {q.shape[1]} and {k.shape[1]}")
    _check_first(q, "Q", "[T, H, D]")
    _check_like(k, "K", q)
    _check_like(v, "V", q)
    _check_tables(cosp, sinp, q)
    _check_cu(cu, q)
    if positions is not None:
        _check_ints(positions, "positions", q.shape[0], q)


# ---------------------------------------------------------------------------
# ops
# ---------------------------------------------------------------------------
@torch.library.custom_op("farope::seq_fwd", mutates_args=())
def _seq_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cosp: torch.Tensor, sinp: torch.Tensor, cu: torch.Tensor,
             positions: Optional[torch.Tensor], causal: bool, has_cls: bool,
             softmax_scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """-> (O [T, H, D], LSE [H, T])."""
    _check_seq(q, k, v, cosp, sinp, cu, positions)
    _check_device(q)
    _lib.require_torch_ops()   # (GPU tensors run the native kernel)


@_seq_fwd.register_fake
def _seq_fwd_fake(q, k, v, cosp, sinp, cu, positions, causal, has_cls, softmax_scale):
    _check_seq(q, k, v, cosp, sinp, cu, positions)
    T, H, D = q.shape
    return q.new_empty((T, H, D)), q.new_empty((H, T), dtype=torch.float32)


@torch.library.custom_op("farope::seq_bwd", mutates_args=())
def _seq_bwd(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
             cosp: torch.Tensor, sinp: torch.Tensor, cu: torch.Tensor, positions: Optional[torch.Tensor], causal: bool,
             has_cls: bool, softmax_scale: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """-> (dQ, dK, dV)."""
    _check_seq(q, k, v, cosp, sinp, cu, positions)
    _check_device(q)
    _lib.require_torch_ops()


@_seq_bwd.register_fake
def _seq_bwd_fake(do, q, k, v, o, lse, cosp, sinp, cu, positions, causal, has_cls, softmax_scale):
    return q.new_empty(tuple(q.shape)), k.new_empty(tuple(k.shape)), v.new_empty(tuple(v.shape))


def _seq_setup_context(ctx, inputs, output):
    q, k, v, cosp, sinp, cu, positions, ctx.causal, ctx.has_cls, ctx.softmax_scale = inputs
    o, lse = output
    ctx.mark_non_differentiable(lse)
    ctx.set_materialize_grads(False)
    ctx.has_positions = positions is not None
    ctx.save_for_backward(q, k, v, o, lse, cosp, sinp, cu, *([positions] if ctx.has_positions else []))


def _seq_backward(ctx, do, _dlse):
    if do is None:
        return (None,) * 10
    q, k, v, o, lse, cosp, sinp, cu, *rest = ctx.saved_tensors
    grads = _seq_bwd(do, q, k, v, o, lse, cosp, sinp, cu, rest[0] if ctx.has_positions else None, ctx.causal, ctx.has_cls,
                     ctx.softmax_scale)
    return (*grads, None, None, None, None, None, None, None)


_seq_fwd.register_autograd(_seq_backward, setup_context=_seq_setup_context)


@torch.library.custom_op("farope::seq_window_fwd", mutates_args=())
def _seq_window_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cosp: torch.Tensor, sinp: torch.Tensor, cu: torch.Tensor,
                    positions: Optional[torch.Tensor], has_cls: bool, softmax_scale: float, window: int,
                    sinks: int) -> tuple[torch.Tensor, torch.Tensor]:
    """-> (O [T, H, D], LSE [H, T])."""
    _check_window(window, sinks)
    _check_seq(q, k, v, cosp, sinp, cu, positions)
    _check_device(q)
    _lib.require_torch_ops()


@_seq_window_fwd.register_fake
def _seq_window_fwd_fake(q, k, v, cosp, sinp, cu, positions, has_cls, softmax_scale, window, sinks):
    _check_window(window, sinks)
    return _seq_fwd_fake(q, k, v, cosp, sinp, cu, positions, True, has_cls, softmax_scale)


@torch.library.custom_op("farope::seq_window_bwd", mutates_args=())
def _seq_window_bwd(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                    cosp: torch.Tensor, sinp: torch.Tensor, cu: torch.Tensor, positions: Optional[torch.Tensor], has_cls: bool,
                    softmax_scale: float, window: int, sinks: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """-> (dQ, dK, dV)."""
    _check_window(window, sinks)
    _check_seq(q, k, v, cosp, sinp, cu, positions)
    _check_device(q)
    _lib.require_torch_ops()


@_seq_window_bwd.register_fake
def _seq_window_bwd_fake(do, q, k, v, o, lse, cosp, sinp, cu, positions, has_cls, softmax_scale, window, sinks):
    return q.new_empty(tuple(q.shape)), k.new_empty(tuple(k.shape)), v.new_empty(tuple(v.shape))


def _seq_window_setup_context(ctx, inputs, output):
    q, k, v, cosp, sinp, cu, positions, ctx.has_cls, ctx.softmax_scale, ctx.window, ctx.sinks = inputs
    o, lse = output
    ctx.mark_non_differentiable(lse)
    ctx.set_materialize_grads(False)
    ctx.has_positions = positions is not None
    ctx.save_for_backward(q, k, v, o, lse, cosp, sinp, cu, *([positions] if ctx.has_positions else []))


def _seq_window_backward(ctx, do, _dlse):
    if do is None:
        return (None,) * 11
    q, k, v, o, lse, cosp, sinp, cu, *rest = ctx.saved_tensors
    grads = _seq_window_bwd(do, q, k, v, o, lse, cosp, sinp, cu, rest[0] if ctx.has_positions else None, ctx.has_cls,
                            ctx.softmax_scale, ctx.window, ctx.sinks)
    return (*grads, None, None, None, None, None, None, None, None)


_seq_window_fwd.register_autograd(_seq_window_backward, setup_context=_seq_window_setup_context)


@torch.library.custom_op("farope::cache_append", mutates_args=("k_cache", "v_cache"))
def _cache_append(k: torch.Tensor, v: torch.Tensor, cosp: torch.Tensor, sinp: torch.Tensor, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, cu: Optional[torch.Tensor],
                  positions: Optional[torch.Tensor], has_cls: bool) -> None:
    _check_append(k, v, cosp, sinp, k_cache, v_cache, page_table, lengths, cu, positions)
    _check_device(k)
    _lib.require_torch_ops()


def _check_append(k, v, cosp, sinp, k_cache, v_cache, page_table, lengths, cu, positions):
    _check_kv(k, v)
    _check_first(k, "K", "[T, Hkv, D]")
    _check_like(v, "V", k)
    _check_tables(cosp, sinp, k)
    _check_cache(k_cache, v_cache, page_table, lengths, k.shape[1], k)
    seqs = page_table.shape[0]
    if cu is not None:
        _check_cu(cu, k)
        if cu.shape[0] != seqs + 1:
            raise ValueError(f"farope: cu_seqlens must hold the page table's {seqs} sequences; got {cu.shape[0]} elements")
    elif k.shape[0] != seqs:
        raise ValueError(f"farope: without cu_seqlens every sequence gets one token; got {k.shape[0]} for {seqs} sequences")
    if positions is not None:
        _check_ints(positions, "positions", k.shape[0], k)


@_cache_append.register_fake
def _cache_append_fake(k, v, cosp, sinp, k_cache, v_cache, page_table, lengths, cu, positions, has_cls):
    _check_append(k, v, cosp, sinp, k_cache, v_cache, page_table, lengths, cu, positions)


@torch.library.custom_op("farope::cache_attn", mutates_args=())
def _cache_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cosp: torch.Tensor, sinp: torch.Tensor,
                page_table: torch.Tensor, lengths: torch.Tensor, positions: Optional[torch.Tensor], has_cls: bool,
                softmax_scale: float) -> torch.Tensor:
    """-> O [B, H, D]."""
    _check_attn(q, k_cache, v_cache, cosp, sinp, page_table, lengths, positions)
    _check_device(q)
    _lib.require_torch_ops()


def _check_attn(q, k_cache, v_cache, cosp, sinp, page_table, lengths, positions):
    _check_first(q, "Q", "[B, H, D]")
    if k_cache.dim() != 4 or k_cache.shape[2] < 1 or q.shape[1] < 1 or q.shape[1] % k_cache.shape[2]:
        raise ValueError("farope: query heads must be a multiple of the cache's key heads; got "
                         f"{tuple(q.shape)} and {tuple(k_cache.shape)}")
    _check_tables(cosp, sinp, q)
    _check_cache(k_cache, v_cache, page_table, lengths, k_cache.shape[2], q)
    if q.shape[0] != page_table.shape[0]:
        raise ValueError(f"farope: one query per sequence: got {q.shape[0]} for {page_table.shape[0]} sequences")
    if positions is not None:
        _check_ints(positions, "positions", q.shape[0], q)


@_cache_attn.register_fake
def _cache_attn_fake(q, k_cache, v_cache, cosp, sinp, page_table, lengths, positions, has_cls, softmax_scale):
    _check_attn(q, k_cache, v_cache, cosp, sinp, page_table, lengths, positions)
    return q.new_empty(tuple(q.shape))


@torch.library.custom_op("farope::cache_attn_window", mutates_args=())
def _cache_attn_window(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cosp: torch.Tensor, sinp: torch.Tensor,
                       page_table: torch.Tensor, lengths: torch.Tensor, positions: Optional[torch.Tensor], has_cls: bool,
                       softmax_scale: float, window: int, sinks: int) -> torch.Tensor:
    """-> O [B, H, D]."""
    _check_window(window, sinks)
    _check_attn(q, k_cache, v_cache, cosp, sinp, page_table, lengths, positions)
    _check_device(q)
    _lib.require_torch_ops()


@_cache_attn_window.register_fake
def _cache_attn_window_fake(q, k_cache, v_cache, cosp, sinp, page_table, lengths, positions, has_cls, softmax_scale, window, sinks):
    _check_window(window, sinks)
    _check_attn(q, k_cache, v_cache, cosp, sinp, page_table, lengths, positions)
    return q.new_empty(tuple(q.shape))


@torch.library.custom_op("farope::cache_tree", mutates_args=())
def _cache_tree(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cosp: torch.Tensor, sinp: torch.Tensor,
                page_table: torch.Tensor, lengths: torch.Tensor, cu: torch.Tensor, tree: Optional[torch.Tensor],
                positions: Optional[torch.Tensor], has_cls: bool, softmax_scale: float) -> torch.Tensor:
    """-> O [T, H, D]."""
    _check_tree(q, k_cache, v_cache, cosp, sinp, page_table, lengths, cu, tree, positions)
    _check_device(q)
    _lib.require_torch_ops()


def _check_tree(q, k_cache, v_cache, cosp, sinp, page_table, lengths, cu, tree, positions):
    _check_first(q, "Q", "[T, H, D]")
    if k_cache.dim() != 4 or k_cache.shape[2] < 1 or q.shape[1] < 1 or q.shape[1] % k_cache.shape[2]:
        raise ValueError("farope: query heads must be a multiple of the cache's key heads; got "
                         f"{tuple(q.shape)} and {tuple(k_cache.shape)}")
    _check_tables(cosp, sinp, q)
    _check_cache(k_cache, v_cache, page_table, lengths, k_cache.shape[2], q)
    _check_cu(cu, q)
    if cu.shape[0] != page_table.shape[0] + 1:
        raise ValueError(f"farope: cu_seqlens must hold the page table's {page_table.shape[0]} sequences; got {cu.shape[0]} elements")
    if tree is not None:
        if tree.dtype != torch.bool:
            raise TypeError(f"farope: tree must be bool; got {tree.dtype}")
        if tree.dim() != 2 or tree.shape[0] != q.shape[0] or (tree.shape[1] > 1 and tree.stride(1) != 1):
            raise ValueError(f"farope: tree must be [T, columns] with T={q.shape[0]}, its rows contiguous; got shape {tuple(tree.shape)}")
        if tree.device != q.device:
            raise RuntimeError("farope: tree must be on the other tensors' device")
    if positions is not None:
        _check_ints(positions, "positions", q.shape[0], q)


@_cache_tree.register_fake
def _cache_tree_fake(q, k_cache, v_cache, cosp, sinp, page_table, lengths, cu, tree, positions, has_cls, softmax_scale):
    _check_tree(q, k_cache, v_cache, cosp, sinp, page_table, lengths, cu, tree, positions)
    return q.new_empty(tuple(q.shape))


_lib.load_torch_ops()   # (their kernels for GPU tensors, as in attention.py)
_seq_fwd_op = torch.ops.farope.seq_fwd.default
_seq_window_fwd_op = torch.ops.farope.seq_window_fwd.default
_append_op = torch.ops.farope.cache_append.default
_attn_op = torch.ops.farope.cache_attn.default
_attn_window_op = torch.ops.farope.cache_attn_window.default
_tree_op = torch.ops.farope.cache_tree.default


# ---------------------------------------------------------------------------
# public entry points
# ---------------------------------------------------------------------------
def _tables(cos_sin):
    cosp, sinp = cos_sin.tables()
    if cosp.is_contiguous() and sinp.is_contiguous():
        return cosp, sinp
    return cosp.contiguous(), sinp.contiguous()


def _scale(head_dim: int) -> float:
    return head_dim ** -0.5 if head_dim else 0.0   # (0 is refused with the other head_dims)


def sdpa_rope_varlen(
    Q: torch.Tensor,
    K: torch.Tensor,
    V: torch.Tensor,
    cos_sin,
    cu_seqlens: torch.Tensor,
    *,
    causal: bool = True,
    has_cls: bool = True,
    positions: Optional[torch.Tensor] = None,
    window: Optional[int] = None,
    sinks: int = 0,
) -> torch.Tensor:
    """Rotary attention within packed sequences, forward and gradients.

    Q: ``[T, H, D]``; K, V: ``[T, Hkv, D]``, H a multiple of Hkv: query head h reads key
    head ``h // (H // Hkv)``.  Any strides; D 32, 64, 128 or 256; bf16, fp16 or fp32 (fp32
    is computed in fp32; under autocast all three are cast to its dtype first).
    cu_seqlens: int32 ``[B + 1]`` on the GPU, the sequences' first tokens in ascending
    order from 0 on, then the end of the last; sequences may be empty.  Tokens behind
    the last sequence come back as zeros, and so do their gradients, whatever they hold.
    The first start counts as 0, the others are cut to 0 .. T; where they do not ascend,
    the rows concerned hold no defined values.
    causal: token i of a sequence sees its tokens 0 .. i, else all of them.  What it does not
    see does not reach O, infinities and NaN included.  (Gradients: an infinity or NaN of Q, K or dO may reach
    a row that it has no part in as 0 * NaN, if it is within 63 tokens of one that has, with a window within 126.)
    window, sinks: of the tokens 0 .. i, token i sees the last ``window`` (at least 1: itself) and those
    below ``sinks`` alone (causal only; without a window ``sinks`` makes no difference).
    positions: int32 ``[T]`` table rows, instead of ``i - has_cls``.

    Returns O ``[T, H, D]`` of Q's dtype.  Gradients come back for Q, K and V.
    """
    if window is not None and not causal:
        raise ValueError("farope: a window is causal")
    cosp, sinp = _tables(cos_sin)
    dtype = Q.dtype
    if torch.is_autocast_enabled():
        comp = _sdpa_comp_dtype(Q)
        Q, K, V = Q.to(comp), K.to(comp), V.to(comp)
    if window is None:
        O = _seq_fwd_op(Q, K, V, cosp, sinp, cu_seqlens, positions, causal, has_cls, _scale(Q.shape[-1]))[0]
    else:
        O = _seq_window_fwd_op(Q, K, V, cosp, sinp, cu_seqlens, positions, has_cls, _scale(Q.shape[-1]), window, sinks)[0]
    return O if O.dtype == dtype else O.to(dtype)


def rope_cache_append(
    K: torch.Tensor,
    V: torch.Tensor,
    cos_sin,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    cu_seqlens: Optional[torch.Tensor] = None,
    has_cls: bool = True,
    positions: Optional[torch.Tensor] = None,
) -> None:
    """Stores new keys, rotated, and values in a paged cache.

    K, V: ``[T, Hkv, D]``, any strides.  k_cache, v_cache: ``[pages, page_rows, Hkv, D]`` of
    K's dtype, written in place; any strides whose rows are 16-byte aligned with contiguous
    channels.  page_table: int32 ``[B, max_pages]``; lengths: int32 ``[B]``, the rows that
    each sequence's cache holds before the call (not changed by it).
    cu_seqlens: int32 ``[B + 1]``, sequence b's new tokens as in ``sdpa_rope_varlen``; without
    it token t is the next one of sequence t.  Token j of sequence b goes to position
    ``lengths[b] + j``, row ``position % page_rows`` of page
    ``page_table[b, position // page_rows]``, and is rotated by table row
    ``position - has_cls``, or by positions[t] (int32 ``[T]``).

    Tokens whose position is past the page table, or whose page number is no page of the
    cache, are not stored, nor are those of a sequence of negative length; no other row
    changes.  No two tokens of a call may share a row.  Not differentiable.
    """
    cosp, sinp = _tables(cos_sin)
    _append_op(K, V, cosp, sinp, k_cache, v_cache, page_table, lengths, cu_seqlens, positions, has_cls)


def sdpa_rope_decode(
    Q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    cos_sin,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    has_cls: bool = True,
    positions: Optional[torch.Tensor] = None,
    window: Optional[int] = None,
    sinks: int = 0,
) -> torch.Tensor:
    """Attention of one new token per sequence over its paged cache.

    Q: ``[B, H, D]`` of the cache's dtype, any strides; caches and page_table as in
    ``rope_cache_append``; lengths: int32 ``[B]``, the rows of each sequence's cache, the
    new token's own among them.  Q is rotated by table row ``lengths[b] - 1 - has_cls``, or by
    positions[b] (int32 ``[B]``).

    window, sinks: the token sees the last ``window`` rows (at least 1: its own) and the first ``sinks`` ones alone,
    as in ``sdpa_rope_varlen``; the rows between them are not read, and their pages may be
    given back.

    How the rows are divided goes by the page table's width (lengths stay on the GPU): for short
    sequences a view of its first columns, as many as they need, is faster.

    Returns O ``[B, H, D]``.  A sequence without rows has O = 0; a length past the page table counts as
    the table's rows, and rows on a page number that is no page of the cache are left out.  No gradients.
    """
    cosp, sinp = _tables(cos_sin)
    args = (Q, k_cache, v_cache, cosp, sinp, page_table, lengths, positions, has_cls, _scale(Q.shape[-1]))
    return _attn_op(*args) if window is None else _attn_window_op(*args, window, sinks)


def sdpa_rope_tree(
    Q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    cos_sin,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    cu_seqlens: torch.Tensor,
    *,
    tree: Optional[torch.Tensor] = None,
    has_cls: bool = True,
    positions: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of several new tokens per sequence over its paged cache: a tree of drafted tokens
    that is to be verified, or, without ``tree``, a chain of tokens, such as a chunk of a prompt.

    The new tokens have been appended (``rope_cache_append`` with the same page_table, lengths,
    cu_seqlens and positions).  Q: ``[T, H, D]`` of the cache's dtype, any strides, packed as
    cu_seqlens (int32 ``[B + 1]``) says; caches and page_table as in ``rope_cache_append``;
    lengths: int32 ``[B]``, the rows of each sequence's cache before the new tokens.
    tree: bool ``[T, columns]``, rows contiguous, less than 2 GiB with what lies between them: token t sees the i-th new token of its sequence where ``tree[t, i]``
    (its ancestors and itself), and every row before them; without it the new tokens up to itself.  What it does not
    see does not reach O, infinities and NaN included.
    Q is rotated by table row ``lengths[b] + j - has_cls`` for the j-th token, or by positions[t] (int32
    ``[T]``): a tree's tokens take the rows of their depths, so that accepted ones (``rope_cache_accept``)
    are where a chain would have put them.

    bf16 and fp16: the rotated Q and the softmax weights are rounded to their type for the products, as in
    ``sdpa_rope_varlen``; ``sdpa_rope_decode`` keeps more of both, so a token's O may differ from its there by
    about the type's rounding.

    Returns O ``[T, H, D]``.  A token that sees no row has O = 0, and so have tokens behind the last
    sequence and those of a sequence of negative length; rows past the page table or on a page number that is no page
    of the cache are left out.  No gradients.
    """
    cosp, sinp = _tables(cos_sin)
    return _tree_op(Q, k_cache, v_cache, cosp, sinp, page_table, lengths, cu_seqlens, tree, positions, has_cls, _scale(Q.shape[-1]))
