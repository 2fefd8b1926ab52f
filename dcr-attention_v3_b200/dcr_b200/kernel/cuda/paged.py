"""Operators of a decode step over a paged key-value cache.

A pool is a pair of tensors ``k_pages`` and ``v_pages`` ``[pages, H_kv, page_size, D]`` (any
strides with contiguous rows, so ``[pages, page_size, H_kv, D]`` pools go in as a transposed
view) and ``page_table [B, max_pages]`` int32 names the pages of each sequence; -1 marks one that
is not mapped. ``page_size`` is any number >= 1, D is 64 or 128, H any multiple of H_kv.

* :func:`paged_append`    - query/key norms, position rotation, append (csrc/dcr_paged_append.cu)
* :func:`paged_attention` - attention of one new token (csrc/dcr_paged_attend.cu)
* :func:`paged_evict`     - eviction by accumulated weight (csrc/dcr_paged_evict.cu)

All take device lengths, so a captured CUDA graph can be replayed while they grow. The reference
has no counterpart: its cache is one contiguous tensor per layer.
:class:`dcr_b200.paged_cache.PagedKVCache` keeps the pool, the tables and the free pages.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from dcr_b200 import _lib
from dcr_b200.kernel.cuda._common import check_dtype, require, workspace

PAGED_HEAD_DIMS = (64, 128)


def _int32(t: torch.Tensor, shape, name: str, device) -> None:
    require(t.dtype == torch.int32 and tuple(t.shape) == tuple(shape) and t.device == device and
            t.is_contiguous(), f"{name} must be a contiguous int32 tensor {tuple(shape)} on {device}")


def _pool(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor):
    """Checks a pool; (dtype code, [pages, H_kv, page_size, D], the six strides)."""
    _lib.require_cuda(k_pages, v_pages, page_table)
    dt = check_dtype(k_pages, "k_pages")
    shape = k_pages.shape
    require(len(shape) == 4 and v_pages.shape == shape and v_pages.dtype == k_pages.dtype and
            v_pages.device == k_pages.device,
            "k_pages and v_pages must be [pages, H_kv, page_size, D] of one shape, dtype and device")
    require(shape[3] in PAGED_HEAD_DIMS, f"head dim must be one of {PAGED_HEAD_DIMS}, got {shape[3]}")
    ks, vs = k_pages.stride(), v_pages.stride()
    require(ks[3] == 1 and vs[3] == 1, "page rows must be contiguous")
    require(page_table.dtype == torch.int32 and page_table.dim() == 2 and
            page_table.device == k_pages.device and page_table.stride(1) == 1,
            "page_table must be [B, max_pages] int32 with contiguous rows, on the pool's device")
    return dt, shape, (ks[0], ks[1], ks[2], vs[0], vs[1], vs[2])


def _slot_table(t: torch.Tensor, dtype: torch.dtype, B: int, H_kv: int, slots: int, name: str,
                device) -> Tuple[int, int]:
    """(batch, head) strides of a per-slot table [B, H_kv, >= slots] with contiguous rows."""
    require(t.dtype == dtype and t.device == device and t.dim() == 3 and t.shape[0] == B and
            t.shape[1] == H_kv and t.shape[2] >= slots and t.stride(2) == 1,
            f"{name} must be {dtype} [{B}, {H_kv}, >= {slots}] with contiguous rows on {device}")
    st = t.stride()
    return st[0], st[1]


def _rows(t: torch.Tensor, T: int, heads: int, D: int, ref: torch.Tensor, name: str):
    """(token, head) strides of [T, heads, D] rows of the pool's dtype."""
    require(t.dim() == 3 and tuple(t.shape) == (T, heads, D) and t.dtype == ref.dtype and
            t.device == ref.device and t.stride(2) == 1,
            f"{name} must be [{T}, {heads}, {D}] {ref.dtype} with contiguous rows on {ref.device}")
    st = t.stride()
    return (st[0] if T > 1 else 0), (st[1] if heads > 1 else 0)


def _call(device: torch.device, name: str, *args) -> None:
    fn = getattr(_lib.load(), name)
    if device.index == torch.cuda.current_device():
        st = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            st = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if st != 0:
        _lib.check(st, name)


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
    dt, (pages, H_kv, page_size, D), strides = _pool(k_pages, v_pages, page_table)
    _lib.require_cuda(q, lengths)
    require(q.dim() == 3, "q must be [B, H, D]")
    B, H = q.shape[0], q.shape[1]
    dev = k_pages.device
    qb, qh = _rows(q, B, H, D, k_pages, "q")
    require(H > 0 and H % H_kv == 0, f"H={H} must be a positive multiple of H_kv={H_kv}")
    require(page_table.shape[0] == B, f"page_table must have {B} rows")
    _int32(lengths, (B,), "lengths", dev)
    require(0 <= window < 1 << 31, "window must be >= 0")
    max_pages = page_table.shape[1]
    slots = max_pages * page_size
    wb = wh = 0
    if weights is not None:
        _lib.require_cuda(weights)
        wb, wh = _slot_table(weights, torch.float32, B, H_kv, slots, "weights", dev)
    if out is None:
        out = torch.empty((B, H, D), dtype=q.dtype, device=dev)
    else:
        require(tuple(out.shape) == (B, H, D) and out.dtype == q.dtype and out.device == dev and
                out.is_contiguous(), f"out must be a contiguous {q.dtype} [{B}, {H}, {D}] on {dev}")
    lse = torch.empty((B, H), dtype=torch.float32, device=dev) if return_lse else None
    if B > 0:
        nbytes = _lib.load().dcr_paged_workspace_bytes(B, H, H_kv, D, slots, weights is not None)
        ws = workspace(dev, nbytes, workspace_buf)
        _call(dev, "dcr_paged_attend", q.data_ptr(), qb, qh, k_pages.data_ptr(),
              v_pages.data_ptr(), dt, *strides, pages, page_size, page_table.data_ptr(),
              page_table.stride(0) if B > 1 else max_pages, max_pages, lengths.data_ptr(), B, H,
              H_kv, D, 1.0 / math.sqrt(D) if scale is None else float(scale), window,
              out.data_ptr(), None if lse is None else lse.data_ptr(),
              None if weights is None else weights.data_ptr(), wb, wh, ws.data_ptr(), ws.numel())
    return (out, lse) if return_lse else out


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
    dt, (pages, H_kv, page_size, D), strides = _pool(k_pages, v_pages, page_table)
    _lib.require_cuda(q, k, v, cos, sin, positions, slots)
    require(q.dim() == 3, "q must be [T, H, D]")
    T, H = q.shape[0], q.shape[1]
    dev = k_pages.device
    require(H > 0 and H % H_kv == 0, f"H={H} must be a positive multiple of H_kv={H_kv}")
    qt, qh = _rows(q, T, H, D, k_pages, "q")
    kt, kh = _rows(k, T, H_kv, D, k_pages, "k")
    vt, vh = _rows(v, T, H_kv, D, k_pages, "v")
    n_seq, max_pages = page_table.shape
    _int32(positions, (T,), "positions", dev)
    _int32(slots, (T,), "slots", dev)
    if seq is not None:
        _lib.require_cuda(seq)
        _int32(seq, (T,), "seq", dev)
    else:
        require(T <= n_seq, f"{T} tokens without seq need as many sequences, got {n_seq}")
    require(cos.dim() == 2 and cos.shape == sin.shape and cos.shape[1] == D and
            cos.shape[0] > 0 and cos.dtype == sin.dtype and
            cos.dtype in (k_pages.dtype, torch.float32) and cos.device == dev and
            sin.device == dev and cos.is_contiguous() and sin.is_contiguous(),
            f"cos and sin must be contiguous [n, {D}] tables of {k_pages.dtype} or float32 on {dev}")
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            require(w.dtype == k_pages.dtype and tuple(w.shape) == (D,) and w.device == dev and
                    w.is_contiguous(), f"{name} must be [{D}] {k_pages.dtype} on {dev}")
    wb = wh = pb = ph = 0
    if weights is not None:
        wb, wh = _slot_table(weights, torch.float32, n_seq, H_kv, max_pages * page_size, "weights", dev)
    if pos is not None:
        pb, ph = _slot_table(pos, torch.int32, n_seq, H_kv, max_pages * page_size, "pos", dev)
    if out is None:
        out = torch.empty((T, H, D), dtype=q.dtype, device=dev)
    else:
        require(tuple(out.shape) == (T, H, D) and out.dtype == q.dtype and out.device == dev and
                out.is_contiguous(), f"out must be a contiguous {q.dtype} [{T}, {H}, {D}] on {dev}")
    if T > 0:
        _call(dev, "dcr_paged_append", q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(),
              vt, vh, None if q_weight is None else q_weight.data_ptr(),
              None if k_weight is None else k_weight.data_ptr(), float(eps), cos.data_ptr(),
              sin.data_ptr(), _lib.DTYPE_CODES[cos.dtype], cos.shape[0], positions.data_ptr(),
              None if seq is None else seq.data_ptr(), slots.data_ptr(), dt, T, H, H_kv, D,
              out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), *strides, pages, page_size,
              page_table.data_ptr(), page_table.stride(0) if n_seq > 1 else max_pages, n_seq,
              max_pages, None if weights is None else weights.data_ptr(), wb, wh,
              None if pos is None else pos.data_ptr(), pb, ph)
    return out


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
    ``[B, H_kv, budget]`` unless given; not the inputs) hold the kept slots' entries."""
    dt, (pages, H_kv, page_size, D), strides = _pool(k_pages, v_pages, page_table)
    _lib.require_cuda(lengths, weights, pos, seen)
    dev = k_pages.device
    B, max_pages = page_table.shape
    slots = max_pages * page_size
    _int32(lengths, (B,), "lengths", dev)
    _int32(seen, (B,), "seen", dev)
    require(0 < budget <= slots, f"budget must be in (0, {slots}], got {budget}")
    require(sinks >= 0 and recent >= 0, "sinks and recent must be >= 0")
    wb, wh = _slot_table(weights, torch.float32, B, H_kv, slots, "weights", dev)
    pb, ph = _slot_table(pos, torch.int32, B, H_kv, slots, "pos", dev)
    if weights_out is None:
        weights_out = torch.empty((B, H_kv, budget), dtype=torch.float32, device=dev)
    if pos_out is None:
        pos_out = torch.empty((B, H_kv, budget), dtype=torch.int32, device=dev)
    wob, woh = _slot_table(weights_out, torch.float32, B, H_kv, budget, "weights_out", dev)
    pob, poh = _slot_table(pos_out, torch.int32, B, H_kv, budget, "pos_out", dev)
    src = torch.empty((B, H_kv, budget), dtype=torch.int32, device=dev)
    lengths_out = torch.empty_like(lengths)
    if B > 0:
        require(weights_out.data_ptr() != weights.data_ptr() and
                pos_out.data_ptr() != pos.data_ptr(),
                "weights_out and pos_out must be other tensors than weights and pos")
        nbytes = _lib.load().dcr_paged_evict_workspace_bytes(B, H_kv, budget)
        ws = workspace(dev, nbytes, workspace_buf)
        _call(dev, "dcr_paged_evict", k_pages.data_ptr(), v_pages.data_ptr(), dt, *strides, pages,
              page_size, page_table.data_ptr(), page_table.stride(0) if B > 1 else max_pages,
              max_pages, lengths.data_ptr(), weights.data_ptr(), wb, wh, pos.data_ptr(), pb, ph,
              seen.data_ptr(), B, H_kv, D, int(budget), int(sinks), int(recent), src.data_ptr(),
              weights_out.data_ptr(), wob, woh, pos_out.data_ptr(), pob, poh,
              lengths_out.data_ptr(), ws.data_ptr(), ws.numel())
    return src, weights_out, pos_out, lengths_out
