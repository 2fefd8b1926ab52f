"""Refusals of the paged serving operators at the C ABI (CPU only). Every call here has one
argument out of order and returns before any CUDA call, so no pointer is followed."""
from __future__ import annotations

import re
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "dcr_b200.h")
NULL, SHAPE, DTYPE, ALIGN, WORKSPACE = 1, 2, 4, 5, 6
BF16, F32 = 0, 2
P = 1 << 20  # an aligned address that is never read
B, H, H_KV, D, PAGES, PAGE, MAX_PAGES = 2, 8, 2, 64, 16, 16, 4


@pytest.fixture(scope="module")
def lib():
    from dcr_b200 import _lib, build
    build.build()
    return _lib.load()


def _names(func):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    args = re.search(r"int %s\s*\(([^)]*)\)" % func, text).group(1)
    return [a.split()[-1].lstrip("*") for a in args.split(",")]


POOL = dict(k_pages=P, v_pages=P, dtype=BF16, num_pages=PAGES, page_size=PAGE, page_table=P,
            table_stride=MAX_PAGES, max_pages=MAX_PAGES, H_kv=H_KV, D=D, stream=None)
for _p in ("k", "v", "kp", "vp"):
    POOL.update({f"{_p}_stride_p": H_KV * PAGE * D, f"{_p}_stride_h": PAGE * D,
                 f"{_p}_stride_s": D, f"{_p}_stride_t": H * D})

ATTEND = dict(POOL, q=P, q_stride_b=H * D, q_stride_h=D, lengths=P, B=B, H=H, scale=0.125,
              window=0, o=P, lse=None, weights=None, w_stride_b=0, w_stride_h=0, workspace=P,
              workspace_bytes=1 << 40)
APPEND = dict(POOL, q=P, k=P, v=P, q_stride_t=H * D, q_stride_h=D, k_stride_h=D, v_stride_h=D,
              q_weight=None, k_weight=None, eps=1e-5, cos=P, sin=P, table_dtype=BF16, n_pos=100,
              positions=P, seq=None, slots=P, T=B, H=H, q_out=P, n_seq=B, weights=None,
              w_stride_b=0, w_stride_h=0, pos=None, p_stride_b=0, p_stride_h=0)
EVICT = dict(POOL, lengths=P, weights=P, w_stride_b=128, w_stride_h=64, pos=P, p_stride_b=128,
             p_stride_h=64, seen=P, B=B, budget=32, sinks=1, recent=1, src_out=P,
             weights_out=2 * P, wo_stride_b=128, wo_stride_h=64, pos_out=2 * P, po_stride_b=128,
             po_stride_h=64, lengths_out=2 * P, workspace=P, workspace_bytes=1 << 40)
LOGITS = dict(logits=P, l_stride_b=100, dtype=F32, B=B, V=100, tokens=P, tokens_are_int64=0,
              t_stride_b=8, L=8, token_lengths=None, prompt_lengths=None, repetition=None,
              presence=None, frequency=None, bias=None, bias_stride_b=0, allowed=None,
              a_stride_b=0, out=P, o_stride_b=100, next_token=P, stream=None)

POOL_REFUSALS = [
    (dict(k_pages=None), NULL), (dict(v_pages=None), NULL), (dict(page_table=None), NULL),
    (dict(dtype=7), DTYPE), (dict(D=96), SHAPE), (dict(H_kv=0), SHAPE), (dict(num_pages=0), SHAPE),
    (dict(page_size=0), SHAPE), (dict(max_pages=0), SHAPE),
    (dict(max_pages=1 << 26, table_stride=1 << 26), SHAPE),  # more than 2^29 slots
    (dict(table_stride=MAX_PAGES - 1), SHAPE),
    (dict(k_pages=P + 8), ALIGN), (dict(v_pages=P + 2), ALIGN)]


def _pool_strides(k, v):
    return [({f"{k}_stride_s": D + 4}, ALIGN), ({f"{v}_stride_p": -D}, SHAPE),
            ({f"{k}_stride_s": D - 8}, SHAPE), ({f"{v}_stride_h": 0}, SHAPE)]


CASES = (
    [("dcr_paged_attend", ATTEND, c, s) for c, s in POOL_REFUSALS + _pool_strides("k", "v") + [
        (dict(q=None), NULL), (dict(lengths=None), NULL), (dict(o=None), NULL), (dict(B=0), SHAPE),
        (dict(H=7), SHAPE), (dict(window=-1), SHAPE), (dict(q=P + 8), ALIGN),
        (dict(o=P + 4), ALIGN), (dict(q_stride_h=D + 1), ALIGN), (dict(q_stride_b=-8), SHAPE),
        (dict(weights=P, w_stride_b=-1), SHAPE), (dict(workspace=None), WORKSPACE),
        (dict(workspace=P + 4), WORKSPACE), (dict(workspace_bytes=0), WORKSPACE)]]
    + [("dcr_paged_append", APPEND, c, s) for c, s in POOL_REFUSALS + _pool_strides("kp", "vp") + [
        (dict(q=None), NULL), (dict(cos=None), NULL), (dict(positions=None), NULL),
        (dict(slots=None), NULL), (dict(q_out=None), NULL), (dict(T=0), SHAPE),
        (dict(n_pos=0), SHAPE), (dict(T=B + 1), SHAPE), (dict(H=7), SHAPE),
        (dict(T=1 << 28, seq=P), SHAPE), (dict(table_dtype=1), DTYPE),
        (dict(k_stride_t=4), ALIGN), (dict(v_stride_h=-D), SHAPE), (dict(sin=P + 8), ALIGN),
        (dict(q_weight=P + 2), ALIGN), (dict(weights=P, w_stride_h=-1), SHAPE),
        (dict(pos=P, p_stride_b=-1), SHAPE)]]
    + [("dcr_paged_evict", EVICT, c, s) for c, s in POOL_REFUSALS + _pool_strides("k", "v") + [
        (dict(lengths=None), NULL), (dict(seen=None), NULL), (dict(src_out=None), NULL),
        (dict(B=0), SHAPE), (dict(B=40000), SHAPE), (dict(budget=0), SHAPE),
        (dict(budget=MAX_PAGES * PAGE + 1), SHAPE), (dict(sinks=-1), SHAPE),
        (dict(recent=-1), SHAPE), (dict(weights_out=P), SHAPE), (dict(pos_out=P), SHAPE),
        (dict(lengths_out=P), SHAPE), (dict(po_stride_h=-1), SHAPE),
        (dict(workspace=None), WORKSPACE), (dict(workspace_bytes=8), WORKSPACE),
        (dict(workspace=P + 1), WORKSPACE), (dict(workspace=P + 2), WORKSPACE)]]
    + [("dcr_process_logits", LOGITS, c, s) for c, s in [
        (dict(logits=None), NULL), (dict(out=None), NULL), (dict(next_token=None), NULL),
        (dict(tokens=None), NULL), (dict(dtype=3), DTYPE), (dict(B=0), SHAPE), (dict(V=0), SHAPE),
        (dict(V=(1 << 30) + 1), SHAPE), (dict(L=-1), SHAPE), (dict(t_stride_b=-1), SHAPE),
        (dict(o_stride_b=99), SHAPE)]])


@pytest.mark.parametrize("func,base,change,status", CASES,
                         ids=[f"{f}-{'-'.join(f'{k}={v}' for k, v in c.items())}"
                              for f, _, c, _ in CASES])
def test_refused(lib, func, base, change, status):
    args = dict(base, **change)
    assert getattr(lib, func)(*[args[n] for n in _names(func)]) == status


def test_workspace_sizes(lib):
    assert lib.dcr_paged_workspace_bytes(B, H, H_KV, D, 64, 0) > 0
    assert lib.dcr_paged_workspace_bytes(B, 7, H_KV, D, 64, 0) == 0
    assert lib.dcr_paged_workspace_bytes(B, H, H_KV, 96, 64, 0) == 0
    assert lib.dcr_paged_evict_workspace_bytes(B, H_KV, 32) == 4 * B * H_KV * 65
    assert lib.dcr_paged_evict_workspace_bytes(B, 0, 32) == 0
