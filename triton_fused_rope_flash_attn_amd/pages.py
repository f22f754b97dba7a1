"""Rows and pages of a paged cache that are there (csrc/cache_pages.hip).

* ``rope_cache_accept``  of the drafted tokens behind a sequence, the accepted ones move up;
* ``rope_cache_fork``    places of a batch continue others' sequences: pages are shared, copied,
                         reserved and freed.

The caches, page tables and lengths are those of ``rope_cache_append`` and
``sdpa_rope_decode`` (sequences.py), and as there all values stay on the GPU: no call waits for the
device, a captured call reads their new values when it is replayed, and none reads or
writes outside its tensors, whatever they are.  There is no CPU fallback.

The reference has no counterpart.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .attention import _check_device
from .sequences import HEAD_DIMS, _check_cache, _check_ints

__all__ = ["rope_cache_accept", "rope_cache_fork"]

MAX_PATH = 2048   # columns of a path


# (CPU and meta tensors; the native kernels make the same checks, with the same exceptions)
def _check_rows(k_cache, v_cache, page_table, lengths):
    if k_cache.dim() != 4 or k_cache.shape[0] < 1 or k_cache.shape[2] < 1:
        raise ValueError(f"farope: the caches must be [pages, page_rows, Hkv, D]; got {tuple(k_cache.shape)}")
    if k_cache.shape[3] not in HEAD_DIMS:
        raise ValueError(f"farope: head_dim must be 32, 64, 128 or 256; got {k_cache.shape[3]}")
    if k_cache.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"farope: unsupported tensor dtype {k_cache.dtype}")
    _check_cache(k_cache, v_cache, page_table, lengths, k_cache.shape[2], k_cache[0])


def _check_accept(k_cache, v_cache, page_table, lengths, path):
    _check_rows(k_cache, v_cache, page_table, lengths)
    seqs = page_table.shape[0]
    if path.dtype != torch.int32:
        raise TypeError(f"farope: path must be int32; got {path.dtype}")
    if path.dim() != 2 or path.shape[0] != seqs or (path.shape[1] > 1 and path.stride(1) != 1):
        raise ValueError(f"farope: path must be [B, columns] with B={seqs}, its rows contiguous; got shape {tuple(path.shape)}")
    if path.shape[1] > MAX_PATH:
        raise ValueError(f"farope: path has at most {MAX_PATH} columns; got {path.shape[1]}")
    if path.device != k_cache.device:
        raise RuntimeError("farope: path must be on the other tensors' device")


def _check_fork(k_cache, v_cache, page_table, lengths, refs, parents, room):
    _check_rows(k_cache, v_cache, page_table, lengths)
    seqs = page_table.shape[0]
    if seqs > 1 and page_table.stride(0) < page_table.shape[1]:
        raise ValueError("farope: the rows of page_table must not overlap")
    _check_ints(refs, "refs", k_cache.shape[0], k_cache)
    _check_ints(parents, "parents", seqs, k_cache)
    if room is not None:
        _check_ints(room, "room", seqs, k_cache)


@torch.library.custom_op("farope::cache_accept", mutates_args=("k_cache", "v_cache"))
def _cache_accept(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                  path: torch.Tensor) -> torch.Tensor:
    """-> the new lengths [B]."""
    _check_accept(k_cache, v_cache, page_table, lengths, path)
    _check_device(k_cache)
    _lib.require_torch_ops()   # (GPU tensors run the native kernel)


@_cache_accept.register_fake
def _cache_accept_fake(k_cache, v_cache, page_table, lengths, path):
    _check_accept(k_cache, v_cache, page_table, lengths, path)
    return lengths.new_empty(tuple(lengths.shape))


@torch.library.custom_op("farope::cache_fork", mutates_args=("k_cache", "v_cache", "page_table", "lengths", "refs"))
def _cache_fork(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                refs: torch.Tensor, parents: torch.Tensor, room: Optional[torch.Tensor]) -> torch.Tensor:
    """-> pages wanted and not there [1]."""
    _check_fork(k_cache, v_cache, page_table, lengths, refs, parents, room)
    _check_device(k_cache)
    _lib.require_torch_ops()


@_cache_fork.register_fake
def _cache_fork_fake(k_cache, v_cache, page_table, lengths, refs, parents, room):
    _check_fork(k_cache, v_cache, page_table, lengths, refs, parents, room)
    return lengths.new_empty((1,))


_accept_op = torch.ops.farope.cache_accept.default
_fork_op = torch.ops.farope.cache_fork.default


def rope_cache_accept(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    path: torch.Tensor,
) -> torch.Tensor:
    """Keeps the accepted ones of the drafted tokens behind each sequence.

    Caches and page_table as in ``rope_cache_append``, the caches written in place; lengths: int32
    ``[B]``, the rows before the drafted tokens (not changed).  path: int32 ``[B, columns]``
    (at most 2048), the accepted drafted tokens of each sequence by their index in the order of the append,
    -1 behind the last: row ``lengths[b] + i`` becomes what row ``lengths[b] + path[b, i]``
    was before the call.  Any order, and a token may come twice.  Keys stay rotated as they are, so a token
    of a tree is to be appended with the position that its depth gives it.

    Returns the new lengths, int32 ``[B]``: lengths plus the number of accepted tokens.  Rows whose
    position is not in the cache (as in ``rope_cache_append``), or whose token's is not, stay as they are, and a sequence
    of negative length does.  No two sequences may share the pages of drafted tokens.  Not differentiable.
    """
    return _accept_op(k_cache, v_cache, page_table, lengths, path)


def rope_cache_fork(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    refs: torch.Tensor,
    parents: torch.Tensor,
    *,
    room: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Each place of the batch continues the sequence of a place: a beam's reordering, the start of
    several continuations of a prompt, the end of a sequence, and the pages that the next tokens need.

    Caches as in ``rope_cache_append``.  page_table: int32 ``[B, max_pages]``, lengths: int32
    ``[B]`` and refs: int32 ``[pages]`` are written in place: an entry of page_table that is no page of
    the cache (-1) holds none, and refs counts the entries that hold each page (what else holds a page
    may be counted too).  A new cache has -1, 0 and 0 throughout.
    parents: int32 ``[B]``: place b continues the sequence of place ``parents[b]``; its own index keeps it as
    it is, a number that is no place (-1) empties it and gives back its pages.
    room: int32 ``[B]``, rows to reserve behind the sequence (without it, 0).

    Whole pages are shared.  The page that the next token falls on, and those behind it, go to the first
    place with that parent, unless something else holds them too; the other places get new pages, with a
    copy of the rows in use.  So does, in place, a sequence whose next row falls on a shared page: where lengths
    were cut back, a call with its own index makes the row safe to write.  New pages are those whose count was 0
    before the call (not those it gives back), the lowest first, in the order of places and
    entries.  Entries that get none are -1, and the tokens there are not stored.

    Returns int32 ``[1]``: the pages that were wanted and not there.  Not differentiable.
    """
    return _fork_op(k_cache, v_cache, page_table, lengths, refs, parents, room)
