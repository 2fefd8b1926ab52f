"""Penalties, bias, grammar mask and the greedy token of a decode step's logits.

The reference's decode loop takes the plain argmax of the logits
(tests/kernel/test_m1_acceptance.py:198); :func:`process_logits` is what a serving loop does
between the LM head and the next token, in one pass over the logits (csrc/dcr_logits.cu).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from dcr_b200 import _lib
from dcr_b200.kernel.cuda._common import check_dtype
from dcr_b200.kernel.cuda.paged import _call, _on_cuda, _refuse


def _per_row(t: Optional[torch.Tensor], B: int, dtype: torch.dtype, name: str, device):
    if t is None:
        return None
    if not (t.dtype is dtype and t.shape == (B,) and t.device == device and t.is_contiguous()):
        _refuse(f"{name} must be a contiguous {dtype} [{B}] on {device}")
    return t.data_ptr()


def process_logits(logits: torch.Tensor, *, tokens: Optional[torch.Tensor] = None,
                   token_lengths: Optional[torch.Tensor] = None,
                   prompt_lengths: Optional[torch.Tensor] = None,
                   repetition: Optional[torch.Tensor] = None,
                   presence: Optional[torch.Tensor] = None,
                   frequency: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(processed logits ``[B, V]`` in the logits' dtype, next token ``[B]`` int64).

    In fp32 and in this order, rounded once: ``x / repetition`` (``x * repetition`` for x <= 0)
    for tokens in the row's history, ``- count * frequency`` and ``- presence`` for those that
    occur after its prompt, ``+ bias``, -inf where ``allowed`` has a clear bit. ``tokens`` ``[B, L]``
    (int32 or int64; negative ids are padding) is the history, ``token_lengths`` ``[B]`` int32 how
    many of each row count (None: all) and ``prompt_lengths`` ``[B]`` int32 how many of these are
    the prompt (None: 0). ``repetition``, ``presence``, ``frequency`` are fp32 ``[B]``, ``bias``
    fp32 ``[V]`` or ``[B, V]``, ``allowed`` int32 ``[B, ceil(V / 32)]`` with token t in bit t % 32
    of word t // 32. The token is the lowest index of the largest returned value among the
    allowed ones (NaN is the largest), -1 where none is allowed. ``out`` may be ``logits``."""
    _on_cuda(logits)
    dtype, dev = logits.dtype, logits.device
    dt = _lib.DTYPE_CODES.get(dtype)
    if dt is None:
        check_dtype(logits, "logits")
    if logits.dim() != 2 or logits.shape[1] == 0 or logits.stride(1) != 1:
        _refuse("logits must be [B, V] with contiguous rows")
    B, V = logits.shape
    L = tok64 = t_stride = 0
    t_ptr = None
    if tokens is not None:
        _on_cuda(tokens)
        if not (tokens.dim() == 2 and tokens.shape[0] == B and tokens.device == dev and
                tokens.dtype in (torch.int32, torch.int64) and
                (tokens.stride(1) == 1 or tokens.shape[1] <= 1)):
            _refuse(f"tokens must be int32 or int64 [{B}, L] with contiguous rows on {dev}")
        L, tok64, t_stride = tokens.shape[1], int(tokens.dtype is torch.int64), tokens.stride(0)
        t_ptr = tokens.data_ptr()
    elif token_lengths is not None or prompt_lengths is not None:
        _refuse("token_lengths and prompt_lengths need tokens")
    n_ptr = _per_row(token_lengths, B, torch.int32, "token_lengths", dev)
    m_ptr = _per_row(prompt_lengths, B, torch.int32, "prompt_lengths", dev)
    r_ptr = _per_row(repetition, B, torch.float32, "repetition", dev)
    p_ptr = _per_row(presence, B, torch.float32, "presence", dev)
    f_ptr = _per_row(frequency, B, torch.float32, "frequency", dev)
    b_ptr, b_stride = None, 0
    if bias is not None:
        if not (bias.dtype is torch.float32 and bias.device == dev and
                bias.shape in ((V,), (B, V)) and (V == 1 or bias.stride(-1) == 1)):
            _refuse(f"bias must be float32 [{V}] or [{B}, {V}] with contiguous rows on {dev}")
        b_ptr, b_stride = bias.data_ptr(), bias.stride(0) if bias.dim() == 2 else 0
    a_ptr, a_stride = None, 0
    if allowed is not None:
        words = (V + 31) // 32
        if not (allowed.dtype is torch.int32 and allowed.device == dev and
                allowed.shape == (B, words) and (words == 1 or allowed.stride(1) == 1)):
            _refuse(f"allowed must be int32 [{B}, {words}] with contiguous rows on {dev}")
        a_ptr, a_stride = allowed.data_ptr(), allowed.stride(0)
    if out is None:
        out = torch.empty((B, V), dtype=dtype, device=dev)
    else:
        if not (out.shape == logits.shape and out.dtype is dtype and out.device == dev and
                out.stride(1) == 1):
            _refuse("out must match logits, with contiguous rows")
        if out.data_ptr() == logits.data_ptr() and out.stride() != logits.stride():
            _refuse("logits processed in place must keep their strides")
    token = torch.empty((B,), dtype=torch.int64, device=dev)
    if B > 0:
        _call(dev, "dcr_process_logits", logits.data_ptr(), logits.stride(0), dt, B, V, t_ptr, tok64,
              t_stride, L, n_ptr, m_ptr, r_ptr, p_ptr, f_ptr, b_ptr, b_stride, a_ptr, a_stride,
              out.data_ptr(), out.stride(0), token.data_ptr())
    return out, token
