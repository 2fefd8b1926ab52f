"""Refusals of the prompt, shared-prefix and rotation operators at the C ABI (CPU only). Every call here
has one argument out of order and returns before any CUDA call, so no pointer is followed."""
from __future__ import annotations

import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_capi_paged import (ALIGN, APPEND, ATTEND, B, D, DTYPE, H, H_KV, NULL, P,  # noqa: E402
                             POOL_REFUSALS, SHAPE, WORKSPACE, _names, _pool_strides, lib)  # noqa: F401

T = 5
PREFILL = dict(ATTEND, q_stride_t=H * D, starts=P, T=T, causal=1, o=P << 1)
SHARED = dict(ATTEND, groups=P, n_groups=1, prefix=P, o=P << 1)
ROTARY_APPEND = dict(APPEND, inv_freq=P, rotated=D, interleaved=0, factor=1.0, q_out=P << 1)
ROTARY = dict(q=P, q_stride_t=H * D, q_stride_h=D, k=P << 1, k_stride_t=H_KV * D, k_stride_h=D, inv_freq=P,
              rotated=D, positions=P, positions_are_int64=0, interleaved=0, factor=1.0, dtype=0, T=T, H=H,
              H_kv=H_KV, D=D, q_out=P << 2, qo_stride_t=H * D, qo_stride_h=D, k_out=P << 3,
              ko_stride_t=H_KV * D, ko_stride_h=D, stream=None)

CASES = (
    [("dcr_paged_prefill", PREFILL, c, s) for c, s in POOL_REFUSALS + _pool_strides("k", "v") + [
        (dict(q=None), NULL), (dict(lengths=None), NULL), (dict(starts=None), NULL), (dict(o=None), NULL),
        (dict(B=0), SHAPE), (dict(T=0), SHAPE), (dict(T=1 << 30), SHAPE), (dict(H=7), SHAPE),
        (dict(window=-1), SHAPE), (dict(window=3, causal=0), SHAPE), (dict(q=P + 8), ALIGN),
        (dict(o=P + 4), ALIGN), (dict(starts=P + 2), ALIGN), (dict(lse=P + 1), ALIGN),
        (dict(q_stride_h=D + 1), ALIGN), (dict(q_stride_t=-8), SHAPE), (dict(o=P + 2 * D), SHAPE),
        (dict(workspace=None), WORKSPACE), (dict(workspace=P + 4), WORKSPACE),
        (dict(workspace_bytes=0), WORKSPACE)]]
    + [("dcr_paged_shared_attend", SHARED, c, s) for c, s in POOL_REFUSALS + _pool_strides("k", "v") + [
        (dict(q=None), NULL), (dict(lengths=None), NULL), (dict(groups=None), NULL), (dict(prefix=None), NULL),
        (dict(o=None), NULL), (dict(B=0), SHAPE), (dict(n_groups=0), SHAPE), (dict(H=7), SHAPE),
        (dict(window=-1), SHAPE), (dict(q=P + 8), ALIGN), (dict(groups=P + 1), ALIGN),
        (dict(prefix=P + 2), ALIGN), (dict(q_stride_h=D + 1), ALIGN), (dict(q_stride_b=-8), SHAPE),
        (dict(workspace=None), WORKSPACE), (dict(workspace_bytes=8), WORKSPACE)]]
    + [("dcr_paged_rotary_append", ROTARY_APPEND, c, s) for c, s in POOL_REFUSALS + _pool_strides("kp", "vp") + [
        (dict(q=None), NULL), (dict(inv_freq=None), NULL), (dict(positions=None), NULL),
        (dict(slots=None), NULL), (dict(q_out=None), NULL), (dict(T=0), SHAPE), (dict(T=B + 1), SHAPE),
        (dict(H=7), SHAPE), (dict(T=1 << 28, seq=P), SHAPE), (dict(rotated=0), SHAPE),
        (dict(rotated=7), SHAPE), (dict(rotated=D + 2), SHAPE), (dict(k_stride_t=4), ALIGN),
        (dict(v_stride_h=-D), SHAPE), (dict(inv_freq=P + 2), ALIGN), (dict(q_weight=P + 2), ALIGN),
        (dict(weights=P, w_stride_h=-1), SHAPE), (dict(pos=P, p_stride_b=-1), SHAPE),
        (dict(q_out=P + 2 * D), SHAPE)]]
    + [("dcr_rotary", ROTARY, c, s) for c, s in [
        (dict(q=None), NULL), (dict(k=None), NULL), (dict(inv_freq=None), NULL), (dict(positions=None), NULL),
        (dict(q_out=None), NULL), (dict(k_out=None), NULL), (dict(dtype=5), DTYPE), (dict(T=0), SHAPE),
        (dict(H=0), SHAPE), (dict(H_kv=0), SHAPE), (dict(D=0), SHAPE), (dict(D=520, rotated=8), SHAPE),
        (dict(D=12, rotated=8), SHAPE), (dict(rotated=0), SHAPE), (dict(rotated=3), SHAPE),
        (dict(rotated=D + 2), SHAPE), (dict(H=1 << 17), SHAPE), (dict(q_stride_t=-8), SHAPE),
        (dict(ko_stride_t=4), ALIGN), (dict(q=P + 8), ALIGN), (dict(positions=P + 2), ALIGN),
        (dict(positions=P + 4, positions_are_int64=1), ALIGN), (dict(qo_stride_h=D - 8), SHAPE),
        (dict(qo_stride_t=0), SHAPE), (dict(q_out=P + 2 * D), SHAPE), (dict(q_out=P << 1), SHAPE),
        (dict(k_out=P), SHAPE), (dict(k_out=(P << 2) + 2 * D), SHAPE)]])


@pytest.mark.parametrize("func,base,change,status", CASES,
                         ids=[f"{f}-{'-'.join(f'{k}={v}' for k, v in c.items())}" for f, _, c, _ in CASES])
def test_refused(lib, func, base, change, status):  # noqa: F811
    args = dict(base, **change)
    assert getattr(lib, func)(*[args[n] for n in _names(func)]) == status


def test_workspace_sizes(lib):  # noqa: F811
    assert lib.dcr_paged_prefill_workspace_bytes(0, T, B, H, H_KV, D) > 0
    assert lib.dcr_paged_prefill_workspace_bytes(0, T, B, 7, H_KV, D) == 0
    assert lib.dcr_paged_prefill_workspace_bytes(0, T, B, H, H_KV, 96) == 0
    assert lib.dcr_paged_shared_workspace_bytes(0, B, 1, H, H_KV, D) > 0
    assert lib.dcr_paged_shared_workspace_bytes(0, B, 0, H, H_KV, D) == 0


def test_frequencies():
    """Scalings of the frequencies against their definitions."""
    import math

    import torch
    from dcr_b200.kernel.cuda import rotary_frequencies
    from dcr_b200.models.llama.attention import llama3_inv_freq
    inv, a = rotary_frequencies(64, 500000.0, scaling="llama3", factor=32.0)
    assert a == 1.0 and torch.allclose(inv, llama3_inv_freq(), rtol=2e-6, atol=0)
    base = 10000.0 ** (-torch.arange(0, 64, 2).double() / 64)
    assert torch.equal(rotary_frequencies(64)[0], base.float())
    assert torch.equal(rotary_frequencies(64, scaling="linear", factor=4.0)[0], (base / 4).float())
    ntk = rotary_frequencies(64, scaling="ntk", factor=8.0)[0].double()
    assert ntk[0] == 1.0 and abs(float(ntk[-1] / base[-1]) - 1 / 8) < 1e-6
    yarn, a = rotary_frequencies(64, scaling="yarn", factor=16.0, original_max_position=4096)
    assert abs(a - (0.1 * math.log(16.0) + 1)) < 1e-12
    ratio = yarn.double() / base
    turns = 4096 * base / (2 * math.pi)
    assert torch.allclose(ratio[turns > 40], torch.ones_like(ratio[turns > 40]), rtol=1e-6)
    assert torch.allclose(ratio[turns < 0.8], torch.full_like(ratio[turns < 0.8], 1 / 16), rtol=1e-6)
    assert (ratio[1:] <= ratio[:-1] + 1e-7).all()
    for bad in (dict(rotated=5), dict(rotated=64, scaling="other"), dict(rotated=64, factor=0.5),
                dict(rotated=64, theta=1.0)):
        with pytest.raises(AssertionError):
            rotary_frequencies(**bad)
