"""Operators of a decode step over a paged key-value cache.

A pool is a pair of tensors ``k_pages`` and ``v_pages`` ``[pages, H_kv, page_size, D]`` (any
strides with contiguous rows, so ``[pages, page_size, H_kv, D]`` pools go in as a transposed
view) and ``page_table [B, max_pages]`` int32 names the pages of each sequence; -1 marks one that
is not mapped. ``page_size`` is any number >= 1, D is 64 or 128, H any multiple of H_kv.

* :func:`paged_append`    - query/key norms, position rotation, append (csrc/dcr_paged_append.cu)
* :func:`paged_rotary_append` - the same, rotated by frequencies in any layout (csrc/dcr_rotary.cu)
* :func:`paged_attention` - attention of one new token (csrc/dcr_paged_attend.cu)
* :func:`paged_prefill`   - attention of many new tokens (csrc/dcr_paged_rows.cu)
* :func:`paged_shared_attention` - attention of one new token where sequences share their first
  pages (csrc/dcr_paged_rows.cu)
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


def paged_prefill_workspace_bytes(T: int, B: int, H: int, H_kv: int, D: int,
                                  dtype: torch.dtype = torch.bfloat16) -> int:
    """Bytes :func:`paged_prefill` needs for T tokens of B sequences."""
    return int(_lib.load().dcr_paged_prefill_workspace_bytes(_lib.DTYPE_CODES[dtype], T, B, H, H_kv, D))


def paged_prefill(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                  page_table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor, *,
                  scale: Optional[float] = None, window: int = 0, causal: bool = True,
                  return_lse: bool = False, out: Optional[torch.Tensor] = None,
                  workspace_buf: Optional[torch.Tensor] = None):
    """Attention of many new tokens per sequence over its cached slots, their own among them.

    q ``[T, H, D]`` (any token and head strides); tokens ``starts[b]`` to ``starts[b + 1] - 1``
    (``starts [B + 1]`` int32 on the device, ascending) are the last of sequence b's ``lengths[b]``
    slots, whose keys and values are in the pages already: a whole prompt, a chunk of one behind
    its history, or drafted tokens to verify. A token sees the slots up to its own (``causal=False``:
    all of the sequence's) and with ``window > 0`` the last ``window`` of these. Returns O ``[T, H,
    D]`` in q's dtype, or (O, lse ``[T, H]`` fp32) with ``return_lse``. Rows of q that belong to no
    sequence are not written: give ``out`` where theirs matter. Statistics and sums are fp32, the
    weights of 16-bit caches enter the second product in 16 bits, O is rounded once."""
    r = _lib.torch_ops().prefill(q, k_pages, v_pages, page_table, lengths, starts, scale, window,
                                 causal, return_lse, out, workspace_buf)
    if type(r) is int:
        _lib.check(r, "dcr_paged_prefill")
    return r


def paged_shared_workspace_bytes(B: int, groups: int, H: int, H_kv: int, D: int,
                                 dtype: torch.dtype = torch.bfloat16) -> int:
    """Bytes :func:`paged_shared_attention` needs."""
    return int(_lib.load().dcr_paged_shared_workspace_bytes(_lib.DTYPE_CODES[dtype], B, groups, H, H_kv,
                                                            D))


def paged_shared_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                           page_table: torch.Tensor, lengths: torch.Tensor, groups: torch.Tensor,
                           prefix: torch.Tensor, *, scale: Optional[float] = None, window: int = 0,
                           return_lse: bool = False, out: Optional[torch.Tensor] = None,
                           workspace_buf: Optional[torch.Tensor] = None):
    """:func:`paged_attention` where groups of sequences hold the same pages in their first slots,
    which are read once for a group.

    Sequences ``groups[p]`` to ``groups[p + 1] - 1`` (``groups [P + 1]`` int32 on the device, from 0
    to B) share the first ``prefix[b]`` slots (``prefix [B]`` int32 on the device) with the group's
    first sequence, whose row of ``page_table`` names the pages; the other slots are looked up in
    the sequence's own row. A group may be one sequence and a prefix 0. Other arguments and the
    result are :func:`paged_attention`'s."""
    r = _lib.torch_ops().shared(q, k_pages, v_pages, page_table, lengths, groups, prefix, scale, window,
                                return_lse, out, workspace_buf)
    if type(r) is int:
        _lib.check(r, "dcr_paged_shared_attend")
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


def paged_rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, inv_freq: torch.Tensor,
                        positions: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                        page_table: torch.Tensor, slots: torch.Tensor, *,
                        seq: Optional[torch.Tensor] = None, interleaved: bool = False,
                        factor: float = 1.0, q_weight: Optional[torch.Tensor] = None,
                        k_weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
                        weights: Optional[torch.Tensor] = None, pos: Optional[torch.Tensor] = None,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`paged_append` with the rotation of :func:`~dcr_b200.kernel.cuda.rotary.rotary`: angles
    from ``inv_freq`` ``[r / 2]`` fp32 instead of tables (any position), the first r elements of a
    head, neighbours paired with ``interleaved``, scaled by ``factor``. Returns the rotated
    queries."""
    r = _lib.torch_ops().rotary_append(q, k, v, inv_freq, positions, k_pages, v_pages, page_table, slots,
                                       seq, interleaved, factor, q_weight, k_weight, eps, weights, pos,
                                       out)
    if type(r) is int:
        _lib.check(r, "dcr_paged_rotary_append")
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
