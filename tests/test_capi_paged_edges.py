"""More refusals of the paged serving operators at the C ABI (CPU only): memory that two writers, or
a reader and a writer, would share, and pointers off their elements' boundary. As in
test_capi_paged.py no pointer is followed."""
from __future__ import annotations

import pytest
from test_capi_paged import (ALIGN, APPEND, ATTEND, B, BF16, D, EVICT, H, H_KV, LOGITS, MAX_PAGES, P,
                             PAGE, SHAPE, _names, lib)  # noqa: F401

SLOTS = MAX_PAGES * PAGE  # 64 a row

# one row for both heads, for both sequences, rows that begin inside one another, sequences inside heads
SHARED = [dict(b=H_KV * SLOTS, h=0), dict(b=0, h=SLOTS), dict(b=H_KV * SLOTS, h=SLOTS - 1),
          dict(b=H_KV * SLOTS - 1, h=SLOTS), dict(b=SLOTS, h=SLOTS), dict(b=SLOTS, h=2 * SLOTS - 1)]
APART = [dict(b=H_KV * SLOTS, h=SLOTS), dict(b=SLOTS, h=B * SLOTS), dict(b=1 << 40, h=SLOTS + 3)]


def _call(lib, func, base, **change):  # noqa: F811
    args = dict(base, **change)
    return getattr(lib, func)(*[args[n] for n in _names(func)])


def _writes(s, slots):
    """Every operator that writes a per-slot table, given one of these strides (scaled to `slots`)."""
    yield "dcr_paged_attend", ATTEND, dict(weights=P, w_stride_b=s["b"], w_stride_h=s["h"])
    yield "dcr_paged_append", APPEND, dict(weights=P, w_stride_b=s["b"], w_stride_h=s["h"])
    yield "dcr_paged_append", APPEND, dict(pos=P, p_stride_b=s["b"], p_stride_h=s["h"])
    yield "dcr_paged_evict", dict(EVICT, budget=slots), dict(wo_stride_b=s["b"], wo_stride_h=s["h"])
    yield "dcr_paged_evict", dict(EVICT, budget=slots), dict(po_stride_b=s["b"], po_stride_h=s["h"])


@pytest.mark.parametrize("s", SHARED, ids=str)
def test_tables_whose_rows_share_elements(lib, s):  # noqa: F811
    for func, base, change in _writes(s, SLOTS):
        assert _call(lib, func, base, **change) == SHAPE, (func, change)


@pytest.mark.parametrize("s", APART, ids=str)
def test_tables_whose_rows_lie_apart_pass_the_checks(lib, s):  # noqa: F811
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses here are not to be followed")
    for func, base, change in _writes(s, SLOTS):
        if func == "dcr_paged_evict":
            change = dict(change, pos_out=P + (1 << 50))
        assert _call(lib, func, base, **change) != SHAPE, (func, change)


DENSE_OUT = dict(wo_stride_b=H_KV * SLOTS, wo_stride_h=SLOTS, po_stride_b=H_KV * SLOTS, po_stride_h=SLOTS)
TABLE = 4 * B * H_KV * SLOTS  # bytes of a dense table


@pytest.mark.parametrize("change", [
    dict(weights_out=P + TABLE - 4 * SLOTS), dict(weights_out=P - TABLE + 4 * SLOTS),
    dict(pos_out=P + 4), dict(pos_out=P - 4),
    dict(weights=5 * P, pos=P, weights_out=P + 8),             # into the positions
    dict(weights=P, pos=5 * P, pos_out=P + 8),                 # into the weights
    dict(weights_out=3 * P, pos_out=3 * P + TABLE // 2),       # into one another
    dict(lengths=9 * P, lengths_out=9 * P + 4 * (B - 1))], ids=str)
def test_evict_outputs_that_reach_into_inputs(lib, change):  # noqa: F811
    base = dict(EVICT, **DENSE_OUT, pos_out=3 * P)
    base.update(w_stride_b=H_KV * SLOTS, w_stride_h=SLOTS, p_stride_b=H_KV * SLOTS, p_stride_h=SLOTS)
    assert _call(lib, "dcr_paged_evict", base, **change) == SHAPE


def test_evict_outputs_between_the_rows_of_inputs_pass(lib):  # noqa: F811
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses here are not to be followed")
    wide = dict(w_stride_b=2 * H_KV * SLOTS, w_stride_h=2 * SLOTS, wo_stride_b=2 * H_KV * SLOTS,
                wo_stride_h=2 * SLOTS, pos=5 * P, pos_out=3 * P)
    for budget, at, fits in ((SLOTS, SLOTS, True), (32, SLOTS + 32, True), (33, SLOTS + 32, False),
                             (SLOTS, SLOTS - 1, False), (32, -32, True), (32, -31, False)):
        got = _call(lib, "dcr_paged_evict", EVICT, **wide, budget=budget, weights_out=P + 4 * at)
        assert (got != SHAPE) == fits, (budget, at)


def _off(func, base, names, by, **kw):
    return [(func, base, dict(kw, **{n: 8 * P + by})) for n in names]


@pytest.mark.parametrize("func,base,change", (
    _off("dcr_paged_attend", ATTEND, ("lengths", "page_table", "lse"), 2)
    + _off("dcr_paged_attend", ATTEND, ("weights",), 2, w_stride_b=H_KV * SLOTS, w_stride_h=SLOTS)
    + _off("dcr_paged_append", APPEND, ("positions", "seq", "slots", "page_table"), 1)
    + _off("dcr_paged_append", APPEND, ("weights",), 2, w_stride_b=H_KV * SLOTS, w_stride_h=SLOTS)
    + _off("dcr_paged_append", APPEND, ("pos",), 3, p_stride_b=H_KV * SLOTS, p_stride_h=SLOTS)
    + _off("dcr_paged_evict", dict(EVICT, pos_out=3 * P), (
        "lengths", "weights", "pos", "seen", "src_out", "weights_out", "pos_out", "lengths_out"), 2)
    + _off("dcr_process_logits", LOGITS, ("logits", "out", "tokens", "token_lengths", "prompt_lengths",
                                          "repetition", "presence", "frequency", "bias", "allowed"), 2)
    + _off("dcr_process_logits", dict(LOGITS, dtype=BF16), ("logits", "out"), 1)
    + _off("dcr_process_logits", LOGITS, ("tokens",), 4, tokens_are_int64=1)
    + _off("dcr_process_logits", LOGITS, ("next_token",), 4)), ids=lambda x: str(x) if isinstance(x, str) else None)
def test_pointers_off_their_elements_boundary(lib, func, base, change):  # noqa: F811
    assert _call(lib, func, base, **change) == ALIGN, change


@pytest.mark.parametrize("change", [
    dict(out=P + 4 * 50), dict(out=P - 4 * 50), dict(out=P + 4),       # reaches into other rows
    dict(out=P, o_stride_b=101),                                       # in place, other rows
    dict(out=P, l_stride_b=0), dict(out=P + 4 * 150, l_stride_b=200),
    dict(dtype=BF16, out=P + 2 * 199)], ids=str)
def test_processed_logits_that_reach_into_the_logits(lib, change):  # noqa: F811
    assert _call(lib, "dcr_process_logits", LOGITS, **change) == SHAPE


@pytest.mark.parametrize("change", [
    dict(), dict(out=P + 4 * 200), dict(dtype=BF16, out=P + 2 * 200), dict(out=P - 4 * 200),
    dict(out=P, l_stride_b=200, o_stride_b=200), dict(out=P + 4 * 100, l_stride_b=200, o_stride_b=200),
    dict(B=1, out=P, o_stride_b=7)], ids=str)
def test_processed_logits_in_place_and_between_the_rows_pass(lib, change):  # noqa: F811
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses here are not to be followed")
    assert _call(lib, "dcr_process_logits", dict(LOGITS, next_token=64 * P), **change) not in (SHAPE, ALIGN)


ROWS = 2 * B * H * D  # bytes of a call's bf16 queries
QKV = dict(q_stride_t=(H + 2 * H_KV) * D, k_stride_t=(H + 2 * H_KV) * D, v_stride_t=(H + 2 * H_KV) * D,
           q=8 * P, k=8 * P + 2 * H * D, v=8 * P + 2 * (H + H_KV) * D)  # slices of packed rows


@pytest.mark.parametrize("func,base,change,fits", [
    ("dcr_paged_attend", ATTEND, dict(q=8 * P, o=8 * P), True),
    ("dcr_paged_attend", ATTEND, dict(q=8 * P, o=8 * P + ROWS), True),
    ("dcr_paged_attend", ATTEND, dict(q=8 * P, o=8 * P + 2 * D), False),
    ("dcr_paged_attend", ATTEND, dict(q=8 * P, o=8 * P - 2 * D), False),
    ("dcr_paged_attend", ATTEND, dict(q=8 * P, o=8 * P, q_stride_b=2 * H * D), False),
    ("dcr_paged_attend", ATTEND, dict(q=8 * P, o=8 * P, q_stride_b=0), False),
    ("dcr_paged_append", APPEND, dict(q=8 * P, q_out=8 * P, k=16 * P, v=32 * P), True),
    ("dcr_paged_append", APPEND, dict(QKV, q_out=64 * P), True),
    ("dcr_paged_append", APPEND, dict(QKV, q_out=8 * P), False),
    ("dcr_paged_append", dict(APPEND, T=1), dict(QKV, q_out=8 * P), True)],
    ids=lambda x: str(x) if isinstance(x, (str, bool)) else None)
def test_outputs_that_reach_into_queries(lib, func, base, change, fits):  # noqa: F811
    import torch
    if fits and torch.cuda.is_available():
        pytest.skip("the addresses here are not to be followed")
    assert (_call(lib, func, base, **change) != SHAPE) == fits
