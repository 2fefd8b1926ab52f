"""Penalties, bias, grammar mask and the greedy token of a decode step's logits.

The reference's decode loop takes the plain argmax of the logits
(tests/kernel/test_m1_acceptance.py:198); :func:`process_logits` is what a serving loop does
between the LM head and the next token, in one pass over the logits (csrc/dcr_logits.cu).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from dcr_b200 import _lib


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
    r = _lib.torch_ops().process_logits(logits, tokens, token_lengths, prompt_lengths, repetition,
                                        presence, frequency, bias, allowed, out)
    if type(r) is int:
        _lib.check(r, "dcr_process_logits")
    return r
