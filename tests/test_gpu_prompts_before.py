"""Prompts of more tokens than their sequence holds slots: tokens before the first slot."""
from __future__ import annotations

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_ref  # noqa: E402
import rows_ref as ref  # noqa: E402
from test_gpu_prompts import DEV, DT, _compare, _gen, _i32, _starts, _status  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("news,lengths", [([50, 3, 9], [20, 3, 0]), ([700, 130], [500, 128]), ([1, 2], [0, 1])])
def test_tokens_before_the_first_slot(dt, causal, news, lengths):
    """With causal they see nothing, without it all slots; whole tiles of the others stay whole."""
    from dcr_b200.kernel.cuda import paged_prefill
    k, v, table = paged_ref.make_pool(lengths, 2, 16, 64, DT[dt], DEV, _gen(1))
    starts = _starts(news)
    q = torch.randn(starts[-1], 8, 64, generator=_gen(2), device=DEV).to(DT[dt])
    o, lse = paged_prefill(q, k, v, table, _i32(lengths), _i32(starts), causal=causal, return_lse=True)
    lo, hi, seq = ref.prefill_limits(starts, lengths, 0, causal)
    want = ref.attend(q, k, v, table[seq], lo, [max(h, 0) for h in hi],
                      weight_unit=0.0 if dt == "f32" else paged_ref.UNIT[DT[dt]])
    _compare(o, lse, want)
    if causal:
        for b, n in enumerate(lengths):
            none = slice(starts[b], starts[b] + max(0, news[b] - n))
            assert (o[none] == 0).all() and (lse[none] == float("-inf")).all()
    assert _status() == 0
