"""Position rotation of query and key heads from frequencies (csrc/dcr_rotary.cu).

:func:`~dcr_b200.kernel.cuda.paged.paged_append` and the decode prologue rotate whole heads in halves by
tables of cosines and sines, as HF apply_rotary_pos_emb
(dcr_attention/models/llama/attention.py:395). :func:`rotary` takes the frequencies instead: halves or neighbours paired, the whole head or its first part, any position
without a table, an amplitude. :func:`rotary_frequencies` makes frequencies and amplitude for the
usual scalings to longer contexts. Arguments are checked in csrc/dcr_torch.cpp, as the paged
operators'.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from dcr_b200 import _lib
from dcr_b200.kernel.cuda._common import require


def rotary(q: torch.Tensor, k: torch.Tensor, inv_freq: torch.Tensor, positions: torch.Tensor, *,
           interleaved: bool = False, factor: float = 1.0, q_out: Optional[torch.Tensor] = None,
           k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, k) with the first ``r = 2 * len(inv_freq)`` elements of every head turned.

    q ``[T, H, D]`` and k ``[T, H_kv, D]`` (any token and head strides, contiguous rows; D a multiple
    of 16 bytes, at most 512), ``inv_freq [r / 2]`` fp32, ``positions [T]`` int32 or int64 of any sign.
    Pairs are (i, i + r/2), or (2i, 2i + 1) with ``interleaved``; the angle is position * inv_freq[i],
    reduced in 64 bits, and both results are scaled by ``factor``. Elements past r are copied. In
    fp32, rounded once. ``q_out`` / ``k_out`` may be q / k themselves (in place: only the r
    elements are read and written); new contiguous tensors are made where they are None."""
    r = _lib.torch_ops().rotary(q, k, inv_freq, positions, interleaved, factor, q_out, k_out)
    if type(r) is int:
        _lib.check(r, "dcr_rotary")
    return r


def rotary_frequencies(rotated: int, theta: float = 10000.0, *, scaling: str = "none",
                       factor: float = 1.0, original_max_position: int = 8192,
                       low_freq_factor: float = 1.0, high_freq_factor: float = 4.0,
                       beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device=None) -> Tuple[torch.Tensor, float]:
    """(inv_freq ``[rotated / 2]`` fp32, amplitude) of theta^(-2i / rotated), stretched ``factor``
    times for contexts longer than ``original_max_position``:

    * "none"; "linear": all frequencies divided by the factor;
    * "ntk": theta raised by factor^(r / (r - 2)), which leaves the first frequency and divides the
      last by the factor;
    * "llama3": wavelengths above original_max_position / low_freq_factor divided, those below
      original_max_position / high_freq_factor kept, a linear blend between;
    * "yarn": frequencies that turn more than beta_fast times within original_max_position kept,
      fewer than beta_slow divided, a linear blend over the index between, and the amplitude 0.1
      ln(factor) + 1."""
    require(rotated > 0 and rotated % 2 == 0, f"rotated must be a positive even number, got {rotated}")
    require(theta > 1.0 and factor >= 1.0, "theta must be above 1 and factor at least 1")
    require(scaling in ("none", "linear", "ntk", "llama3", "yarn"), f"unknown scaling {scaling!r}")
    i = torch.arange(0, rotated, 2, dtype=torch.float64)
    amplitude = 1.0
    if scaling == "ntk" and rotated > 2:
        theta = theta * factor ** (rotated / (rotated - 2))
    inv = theta ** (-i / rotated)
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "llama3":
        turns = original_max_position * inv / (2 * math.pi)  # within the original context
        keep = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0, 1)
        inv = inv * (keep + (1 - keep) / factor)
    elif scaling == "yarn":
        def index_of(turns):  # the (fractional) frequency that turns so often
            return rotated * math.log(original_max_position / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(index_of(beta_fast)), 0), min(math.ceil(index_of(beta_slow)), rotated - 1)
        keep = 1 - ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        inv = inv * (keep + (1 - keep) / factor)
        amplitude = 0.1 * math.log(factor) + 1.0
    return inv.float().to(device), amplitude
