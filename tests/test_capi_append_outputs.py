"""Outputs of the appends that reach into the keys and values beside them are refused at the C ABI (CPU
only: the addresses are not followed)."""
from __future__ import annotations

import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_capi_paged import APPEND, B, D, H, H_KV, _names, lib  # noqa: E402,F401
from test_capi_paged_edges import P, QKV  # noqa: E402
from test_capi_prompts import ROTARY_APPEND  # noqa: E402

OVERLAP = 10
OUT = 2 * B * H * D  # bytes of a call's bf16 outputs
APART = dict(q=8 * P, k=16 * P, v=32 * P)
KV = 2 * ((B - 1) * H * D + H_KV * D)  # bytes that the keys span: rows H * D elements apart


def _refused(lib, func, base, change):  # noqa: F811
    args = dict(base, **change)
    return getattr(lib, func)(*[args[n] for n in _names(func)]) == OVERLAP


CASES = [
    (dict(APART, q_out=64 * P), False),
    (dict(APART, q_out=8 * P), False),                 # the queries themselves
    (dict(APART, q_out=16 * P), True),                 # the keys'
    (dict(APART, q_out=32 * P), True),                 # the values'
    (dict(APART, q_out=16 * P + KV - 2 * D), True),    # their last row's
    (dict(APART, q_out=32 * P - OUT + 2 * D), True),   # their first's
    (dict(APART, q_out=16 * P + KV), False),
    (dict(APART, q_out=32 * P - OUT), False),
    (dict(QKV, q_out=64 * P), False),                  # slices of packed rows
    (dict(QKV, q_out=8 * P + 2 * (H + 2 * H_KV) * D * B), False),
    (dict(APART, q_out=16 * P, k_stride_t=0, k_stride_h=0), True)]


def _check(lib, func, base, change, refused):  # noqa: F811
    import torch
    if not refused and torch.cuda.is_available():
        pytest.skip("the addresses here are not to be followed")
    assert _refused(lib, func, base, change) == refused


@pytest.mark.parametrize("change,refused", CASES, ids=str)
def test_rotary_append(lib, change, refused):  # noqa: F811
    _check(lib, "dcr_paged_rotary_append", ROTARY_APPEND, change, refused)


@pytest.mark.parametrize("change,refused", CASES, ids=str)
def test_append(lib, change, refused):  # noqa: F811
    _check(lib, "dcr_paged_append", APPEND, change, refused)
