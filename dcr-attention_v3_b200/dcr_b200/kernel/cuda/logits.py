"""Penalties, bias, grammar mask and the greedy token of a decode step's logits.

The reference's decode loop takes the plain argmax of the logits
(tests/kernel/test_m1_acceptance.py:198); :func:`process_logits` is what a serving loop does
between the LM head and the next token, in one pass over the logits (csrc/dcr_logits.cu).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from dcr_b200 import _lib
from dcr_b200.kernel.cuda._common import check_dtype, require, workspace
from dcr_b200.kernel.cuda.paged import _call


def _per_row(t: Optional[torch.Tensor], B: int, dtype: torch.dtype, name: str, device):
    if t is None:
        return None
    require(t.dtype == dtype and tuple(t.shape) == (B,) and t.device == device and
            t.is_contiguous(), f"{name} must be a contiguous {dtype} [{B}] on {device}")
    return t.data_ptr()


def process_logits(logits: torch.Tensor, *, tokens: Optional[torch.Tensor] = None,
                   token_lengths: Optional[torch.Tensor] = None,
                   prompt_lengths: Optional[torch.Tensor] = None,
                   repetition: Optional[torch.Tensor] = None,
                   presence: Optional[torch.Tensor] = None,
                   frequency: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None,
                   workspace_buf: Optional[torch.Tensor] = None
                   ) -> Tuple[torch.Tensor, torch.Tensor]:
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
    _lib.require_cuda(logits)
    dt = check_dtype(logits, "logits")
    require(logits.dim() == 2 and logits.shape[1] > 0 and logits.stride(1) == 1,
            "logits must be [B, V] with contiguous rows")
    B, V = logits.shape
    dev = logits.device
    L = tok64 = t_stride = 0
    if tokens is not None:
        _lib.require_cuda(tokens)
        require(tokens.dim() == 2 and tokens.shape[0] == B and tokens.device == dev and
                tokens.dtype in (torch.int32, torch.int64) and
                (tokens.stride(1) == 1 or tokens.shape[1] <= 1),
                f"tokens must be int32 or int64 [{B}, L] with contiguous rows on {dev}")
        L, tok64, t_stride = tokens.shape[1], int(tokens.dtype == torch.int64), tokens.stride(0)
    else:
        require(token_lengths is None and prompt_lengths is None,
                "token_lengths and prompt_lengths need tokens")
    n_ptr = _per_row(token_lengths, B, torch.int32, "token_lengths", dev)
    m_ptr = _per_row(prompt_lengths, B, torch.int32, "prompt_lengths", dev)
    r_ptr = _per_row(repetition, B, torch.float32, "repetition", dev)
    p_ptr = _per_row(presence, B, torch.float32, "presence", dev)
    f_ptr = _per_row(frequency, B, torch.float32, "frequency", dev)
    b_ptr, b_stride = None, 0
    if bias is not None:
        require(bias.dtype == torch.float32 and bias.device == dev and
                tuple(bias.shape) in ((V,), (B, V)) and
                (V == 1 or bias.stride(-1) == 1),
                f"bias must be float32 [{V}] or [{B}, {V}] with contiguous rows on {dev}")
        b_ptr, b_stride = bias.data_ptr(), bias.stride(0) if bias.dim() == 2 else 0
    a_ptr, a_stride = None, 0
    if allowed is not None:
        words = (V + 31) // 32
        require(allowed.dtype == torch.int32 and allowed.device == dev and
                tuple(allowed.shape) == (B, words) and (words == 1 or allowed.stride(1) == 1),
                f"allowed must be int32 [{B}, {words}] with contiguous rows on {dev}")
        a_ptr, a_stride = allowed.data_ptr(), allowed.stride(0)
    if out is None:
        out = torch.empty((B, V), dtype=logits.dtype, device=dev)
    else:
        require(out.shape == logits.shape and out.dtype == logits.dtype and out.device == dev and
                out.stride(1) == 1, "out must match logits, with contiguous rows")
        require(out.data_ptr() != logits.data_ptr() or out.stride() == logits.stride(),
                "logits processed in place must keep their strides")
    token = torch.empty((B,), dtype=torch.int64, device=dev)
    if B > 0:
        nbytes = _lib.load().dcr_logits_workspace_bytes(B, V, L)
        ws = workspace(dev, nbytes, workspace_buf)
        _call(dev, "dcr_process_logits", logits.data_ptr(), logits.stride(0), dt, B, V,
              None if tokens is None else tokens.data_ptr(), tok64, t_stride, L, n_ptr, m_ptr, r_ptr,
              p_ptr, f_ptr, b_ptr, b_stride, a_ptr, a_stride, out.data_ptr(), out.stride(0),
              token.data_ptr(), ws.data_ptr(), ws.numel())
    return out, token
