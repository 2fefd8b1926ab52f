"""Operators of a decode step over a paged key-value cache.

A pool is a pair of tensors ``k_pages`` and ``v_pages`` ``[pages, H_kv, page_size, D]`` (any
strides with contiguous rows, so ``[pages, page_size, H_kv, D]`` pools go in as a transposed
view) and ``page_table [B, max_pages]`` int32 names the pages of each sequence; -1 marks one that
is not mapped. ``page_size`` is any number >= 1, D is 64 or 128, H any multiple of H_kv.

* :func:`paged_append`    - query/key norms, position rotation, append (csrc/dcr_paged_append.cu)
* :func:`paged_attention` - attention of one new token (csrc/dcr_paged_attend.cu)
* :func:`paged_evict`     - eviction by accumulated weight (csrc/dcr_paged_evict.cu)

All take device lengths, so a captured CUDA graph can be replayed while they grow. Arguments are
checked in csrc/dcr_torch.cpp: shapes, dtypes, layouts and values raise AssertionError, tensors
that are not on a CUDA device RuntimeError. The reference has no counterpart: its cache is one
contiguous tensor per layer.
:class:`dcr_b200.paged_cache.PagedKVCache` keeps the pool, the tables and the free pages.
"""
from __future__ import annotations

from typing import Optional

import torch

from dcr_b200 import _lib

PAGED_HEAD_DIMS = (64, 128)


def paged_workspace_bytes(B: int, H: int, H_kv: int, D: int, max_slots: int,
                          with_weights: bool = False) -> int:
    """Bytes :func:`paged_attention` needs for this shape (max_slots = max_pages * page_size)."""
    return int(_lib.load().dcr_paged_workspace_bytes(B, H, H_kv, D, max_slots, int(with_weights)))


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    page_table: torch.Tensor, lengths: torch.Tensor, *,
                    scale: Optional[float] = None, window: int = 0,
                    weights: Optional[torch.Tensor] = None, return_lse: bool = False,
                    out: Optional[torch.Tensor] = None,
                    workspace_buf: Optional[torch.Tensor] = None):
    """Attention of one new token per sequence over its cached slots.

    q ``[B, H, D]`` (any batch and head strides), lengths ``[B]`` int32 on the device (0: the
    row is 0), scale 1/sqrt(D) by default; window > 0 attends to the last ``window`` slots.
    ``weights`` (fp32 ``[B, H_kv, >= max_pages * page_size]``) is increased in place by each
    slot's attention weight, summed over the KV head's query heads, the measure that
    :func:`paged_evict` goes by. Returns O ``[B, H, D]`` in q's dtype, or (O, lse ``[B, H]``
    fp32) with ``return_lse``. Softmax statistics and sums are fp32, O is rounded once."""
    r = _lib.torch_ops().attend(q, k_pages, v_pages, page_table, lengths, scale, window, weights,
                                return_lse, out, workspace_buf)
    if type(r) is int:
        _lib.check(r, "dcr_paged_attend")
    return r


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
                 sin: torch.Tensor, positions: torch.Tensor, k_pages: torch.Tensor,
                 v_pages: torch.Tensor, page_table: torch.Tensor, slots: torch.Tensor, *,
                 seq: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
                 weights: Optional[torch.Tensor] = None, pos: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Norms, rotation and append of T tokens in one launch; returns the rotated queries.

    q ``[T, H, D]``, k and v ``[T, H_kv, D]`` (any token and head strides: slices of packed
    projections go in as they are). Each query and key row is RMS-normed over D with ``q_weight``
    / ``k_weight`` ``[D]`` (None: no norm), rotated with row ``positions[t]`` of ``cos`` and
    ``sin`` ``[n, D]`` (the model dtype or fp32; HF apply_rotary_pos_emb), in fp32, rounded once.
    Keys and values are written to slot ``slots[t]`` of sequence ``seq[t]`` (None: token t is
    sequence t's; a negative slot: not written). ``weights`` / ``pos`` (per-slot tables of a cache
    under eviction, fp32 / int32 ``[B, H_kv, slots]``) get 0 / ``positions[t]`` there."""
    r = _lib.torch_ops().append(q, k, v, cos, sin, positions, k_pages, v_pages, page_table, slots,
                                seq, q_weight, k_weight, eps, weights, pos, out)
    if type(r) is int:
        _lib.check(r, "dcr_paged_append")
    return r


def paged_evict(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                lengths: torch.Tensor, weights: torch.Tensor, pos: torch.Tensor,
                seen: torch.Tensor, budget: int, *, sinks: int = 0, recent: int = 0,
                weights_out: Optional[torch.Tensor] = None, pos_out: Optional[torch.Tensor] = None,
                workspace_buf: Optional[torch.Tensor] = None):
    """Keeps ``budget`` slots of every sequence and KV head that holds more; (src, weights_out,
    pos_out, lengths_out).

    Protected slots stay first (``pos`` below ``sinks``, or among the last ``recent`` of the
    ``seen[b]`` positions so far), then those of the largest accumulated ``weights``; equal ones
    go by the lower slot, NaN ranks highest. Kept rows at or past the budget move, in place and in
    slot order, into the evicted slots before it. ``src [B, H_kv, budget]`` int32 is the slot each
    kept row came from (-1 past the new length); ``weights_out`` and ``pos_out`` (new tensors
    ``[B, H_kv, budget]`` unless given; not the inputs) hold the kept slots' entries. Every page
    below a length must be mapped: a row that would come from or go to one that is not stays where
    it is, its new slot is -1 in ``src`` and the device status is set."""
    r = _lib.torch_ops().evict(k_pages, v_pages, page_table, lengths, weights, pos, seen, budget,
                               sinks, recent, weights_out, pos_out, workspace_buf)
    if type(r) is int:
        _lib.check(r, "dcr_paged_evict")
    return r
