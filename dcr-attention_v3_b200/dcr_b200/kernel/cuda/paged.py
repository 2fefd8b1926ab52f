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
from functools import lru_cache
from typing import Optional, Tuple

import torch

from dcr_b200 import _lib
from dcr_b200.kernel.cuda._common import check_dtype, workspace

PAGED_HEAD_DIMS = (64, 128)


# The checks run on every step of a decode loop, so their messages are only formatted on failure.
def _refuse(msg: str) -> None:
    raise AssertionError(msg)


def _on_cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if not t.is_cuda:
            _lib.require_cuda(t)


def _int32(t: torch.Tensor, n: int, name: str, device) -> int:
    """The pointer of a contiguous int32 [n]."""
    if not (t.dtype is torch.int32 and t.shape == (n,) and t.device == device and
            t.is_contiguous()):
        _refuse(f"{name} must be a contiguous int32 tensor [{n}] on {device}")
    return t.data_ptr()


def _pool(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor):
    """Checks a pool; (dtype code, [pages, H_kv, page_size, D], the six strides, device)."""
    _on_cuda(k_pages, v_pages, page_table)
    dtype, shape, device = k_pages.dtype, k_pages.shape, k_pages.device
    dt = _lib.DTYPE_CODES.get(dtype)
    if dt is None:
        check_dtype(k_pages, "k_pages")
    if not (len(shape) == 4 and v_pages.shape == shape and v_pages.dtype is dtype and
            v_pages.device == device):
        _refuse("k_pages and v_pages must be [pages, H_kv, page_size, D] of one shape, dtype and device")
    if shape[3] not in PAGED_HEAD_DIMS:
        _refuse(f"head dim must be one of {PAGED_HEAD_DIMS}, got {shape[3]}")
    ks, vs = k_pages.stride(), v_pages.stride()
    if not (ks[3] == 1 and vs[3] == 1):
        _refuse("page rows must be contiguous")
    if not (page_table.dtype is torch.int32 and page_table.dim() == 2 and
            page_table.device == device and page_table.stride(1) == 1):
        _refuse("page_table must be [B, max_pages] int32 with contiguous rows, on the pool's device")
    return dt, shape, (ks[0], ks[1], ks[2], vs[0], vs[1], vs[2]), device


def _slot_table(t: torch.Tensor, dtype: torch.dtype, B: int, H_kv: int, slots: int, name: str,
                device) -> Tuple[int, int, int]:
    """(pointer, batch stride, head stride) of a per-slot table [B, H_kv, >= slots]."""
    _on_cuda(t)
    shape, st = t.shape, t.stride()
    if not (t.dtype is dtype and t.device == device and len(shape) == 3 and shape[0] == B and
            shape[1] == H_kv and shape[2] >= slots and st[2] == 1):
        _refuse(f"{name} must be {dtype} [{B}, {H_kv}, >= {slots}] with contiguous rows on {device}")
    return t.data_ptr(), st[0], st[1]


def _rows(t: torch.Tensor, shape, dtype: torch.dtype, device, name: str) -> Tuple[int, int, int]:
    """(pointer, token stride, head stride) of rows [tokens, heads, D]."""
    _on_cuda(t)
    st = t.stride()
    if not (t.shape == shape and t.dtype is dtype and t.device == device and st[2] == 1):
        _refuse(f"{name} must be {list(shape)} {dtype} with contiguous rows on {device}")
    return t.data_ptr(), (st[0] if shape[0] > 1 else 0), (st[1] if shape[1] > 1 else 0)


def _output(out: Optional[torch.Tensor], shape, dtype: torch.dtype, device) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if not (out.shape == shape and out.dtype is dtype and out.device == device and
            out.is_contiguous()):
        _refuse(f"out must be a contiguous {dtype} {list(shape)} on {device}")
    return out


def _call(device: torch.device, name: str, *args) -> None:
    fn = getattr(_lib.load(), name)
    index = device.index
    if index == torch._C._cuda_getDevice():
        st = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            st = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if st != 0:
        _lib.check(st, name)


@lru_cache(maxsize=1024)
def _bytes(name: str, device_index: int, *shape: int) -> int:
    with torch.cuda.device(device_index):
        return int(getattr(_lib.load(), name)(*shape))


def _scratch(device: torch.device, nbytes: int, ws: Optional[torch.Tensor]) -> torch.Tensor:
    if ws is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    return workspace(device, nbytes, ws)


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
    dt, (pages, H_kv, page_size, D), strides, dev = _pool(k_pages, v_pages, page_table)
    _on_cuda(q, lengths)
    if q.dim() != 3:
        _refuse("q must be [B, H, D]")
    B, H, _ = q.shape
    q_ptr, qb, qh = _rows(q, (B, H, D), k_pages.dtype, dev, "q")
    if H <= 0 or H % H_kv != 0:
        _refuse(f"H={H} must be a positive multiple of H_kv={H_kv}")
    n_tables, max_pages = page_table.shape
    if n_tables != B:
        _refuse(f"page_table must have {B} rows")
    n_ptr = _int32(lengths, B, "lengths", dev)
    if not 0 <= window < 1 << 31:
        _refuse("window must be >= 0")
    slots = max_pages * page_size
    w_ptr, wb, wh = None, 0, 0
    if weights is not None:
        w_ptr, wb, wh = _slot_table(weights, torch.float32, B, H_kv, slots, "weights", dev)
    out = _output(out, (B, H, D), q.dtype, dev)
    lse = torch.empty((B, H), dtype=torch.float32, device=dev) if return_lse else None
    if B > 0:
        ws = _scratch(dev, _bytes("dcr_paged_workspace_bytes", dev.index, B, H, H_kv, D, slots,
                                  0 if weights is None else 1), workspace_buf)
        _call(dev, "dcr_paged_attend", q_ptr, qb, qh, k_pages.data_ptr(), v_pages.data_ptr(), dt,
              *strides, pages, page_size, page_table.data_ptr(),
              page_table.stride(0) if B > 1 else max_pages, max_pages, n_ptr, B, H, H_kv, D,
              1.0 / math.sqrt(D) if scale is None else float(scale), window, out.data_ptr(),
              None if lse is None else lse.data_ptr(), w_ptr, wb, wh, ws.data_ptr(), ws.numel())
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
    dt, (pages, H_kv, page_size, D), strides, dev = _pool(k_pages, v_pages, page_table)
    _on_cuda(q, cos, sin, positions, slots)
    dtype = k_pages.dtype
    if q.dim() != 3:
        _refuse("q must be [T, H, D]")
    T, H, _ = q.shape
    if H <= 0 or H % H_kv != 0:
        _refuse(f"H={H} must be a positive multiple of H_kv={H_kv}")
    q_ptr, qt, qh = _rows(q, (T, H, D), dtype, dev, "q")
    k_ptr, kt, kh = _rows(k, (T, H_kv, D), dtype, dev, "k")
    v_ptr, vt, vh = _rows(v, (T, H_kv, D), dtype, dev, "v")
    n_seq, max_pages = page_table.shape
    p_ptr = _int32(positions, T, "positions", dev)
    s_ptr = _int32(slots, T, "slots", dev)
    seq_ptr = None
    if seq is not None:
        _on_cuda(seq)
        seq_ptr = _int32(seq, T, "seq", dev)
    elif T > n_seq:
        _refuse(f"{T} tokens without seq need as many sequences, got {n_seq}")
    table_dtype, table_shape = cos.dtype, cos.shape
    if not (len(table_shape) == 2 and sin.shape == table_shape and table_shape[1] == D and
            table_shape[0] > 0 and sin.dtype is table_dtype and
            (table_dtype is dtype or table_dtype is torch.float32) and cos.device == dev and
            sin.device == dev and cos.is_contiguous() and sin.is_contiguous()):
        _refuse(f"cos and sin must be contiguous [n, {D}] tables of {dtype} or float32 on {dev}")
    norm_ptrs = [None, None]
    for i, w in enumerate((q_weight, k_weight)):
        if w is not None:
            if not (w.dtype is dtype and w.shape == (D,) and w.device == dev and w.is_contiguous()):
                _refuse(f"{'k_weight' if i else 'q_weight'} must be [{D}] {dtype} on {dev}")
            norm_ptrs[i] = w.data_ptr()
    w_ptr = pos_ptr = None
    wb = wh = pb = ph = 0
    if weights is not None:
        w_ptr, wb, wh = _slot_table(weights, torch.float32, n_seq, H_kv, max_pages * page_size,
                                    "weights", dev)
    if pos is not None:
        pos_ptr, pb, ph = _slot_table(pos, torch.int32, n_seq, H_kv, max_pages * page_size, "pos", dev)
    out = _output(out, (T, H, D), dtype, dev)
    if T > 0:
        _call(dev, "dcr_paged_append", q_ptr, qt, qh, k_ptr, kt, kh, v_ptr, vt, vh, *norm_ptrs,
              float(eps), cos.data_ptr(), sin.data_ptr(), _lib.DTYPE_CODES[table_dtype],
              table_shape[0], p_ptr, seq_ptr, s_ptr, dt, T, H, H_kv, D, out.data_ptr(),
              k_pages.data_ptr(), v_pages.data_ptr(), *strides, pages, page_size,
              page_table.data_ptr(), page_table.stride(0) if n_seq > 1 else max_pages, n_seq,
              max_pages, w_ptr, wb, wh, pos_ptr, pb, ph)
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
    dt, (pages, H_kv, page_size, D), strides, dev = _pool(k_pages, v_pages, page_table)
    _on_cuda(lengths, seen)
    B, max_pages = page_table.shape
    slots = max_pages * page_size
    n_ptr = _int32(lengths, B, "lengths", dev)
    seen_ptr = _int32(seen, B, "seen", dev)
    if not 0 < budget <= slots:
        _refuse(f"budget must be in (0, {slots}], got {budget}")
    if not (0 <= sinks < 1 << 31 and 0 <= recent < 1 << 31):
        _refuse("sinks and recent must be >= 0")
    w_ptr, wb, wh = _slot_table(weights, torch.float32, B, H_kv, slots, "weights", dev)
    p_ptr, pb, ph = _slot_table(pos, torch.int32, B, H_kv, slots, "pos", dev)
    if weights_out is None:
        weights_out = torch.empty((B, H_kv, budget), dtype=torch.float32, device=dev)
    if pos_out is None:
        pos_out = torch.empty((B, H_kv, budget), dtype=torch.int32, device=dev)
    wo_ptr, wob, woh = _slot_table(weights_out, torch.float32, B, H_kv, budget, "weights_out", dev)
    po_ptr, pob, poh = _slot_table(pos_out, torch.int32, B, H_kv, budget, "pos_out", dev)
    src = torch.empty((B, H_kv, budget), dtype=torch.int32, device=dev)
    lengths_out = torch.empty((B,), dtype=torch.int32, device=dev)
    if B > 0:
        if wo_ptr == w_ptr or po_ptr == p_ptr:
            _refuse("weights_out and pos_out must be other tensors than weights and pos")
        ws = _scratch(dev, _bytes("dcr_paged_evict_workspace_bytes", dev.index, B, H_kv, int(budget)),
                      workspace_buf)
        _call(dev, "dcr_paged_evict", k_pages.data_ptr(), v_pages.data_ptr(), dt, *strides, pages,
              page_size, page_table.data_ptr(), page_table.stride(0) if B > 1 else max_pages,
              max_pages, n_ptr, w_ptr, wb, wh, p_ptr, pb, ph, seen_ptr, B, H_kv, D, budget, sinks,
              recent, src.data_ptr(), wo_ptr, wob, woh, po_ptr, pob, poh, lengths_out.data_ptr(),
              ws.data_ptr(), ws.numel())
    return src, weights_out, pos_out, lengths_out
