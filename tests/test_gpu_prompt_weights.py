"""Attention weights of prompts in a cache with a budget: what is evicted does not depend on where a prompt is
cut into chunks."""
from __future__ import annotations

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_paged_prompts import DEV, _model, _tokens  # noqa: E402

pytestmark = pytest.mark.gpu


def _feed(paged, chunks, decode=0):
    """Sequence 0's prompt in these chunks, beside a short one that goes on decoding; the cache."""
    cache = paged.new_cache(2, 60, 96, page_size=8, budget=24, sinks=1, recent=2, slack=16)
    paged.prefill([_tokens(10, 1), _tokens(3, 2)], cache)
    for t in range(decode):
        paged.step(torch.tensor([t, 5], device=DEV), cache)
    tokens = _tokens(sum(chunks), 3)
    for n in chunks:
        paged.prefill([tokens[:n], []], cache)
        tokens = tokens[n:]
    return cache


@pytest.mark.parametrize("decode", [0, 4])
@pytest.mark.parametrize("chunks", [(16, 4, 1), (5, 12, 4), (20, 1), (1,) * 21])
def test_chunks_weigh_as_the_whole_prompt(decode, chunks):
    """31 or 35 slots, between the budget of 24 and the 40 that are evicted from: chunks that end over the budget
    counted their last tokens too."""
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=256)
    whole, cut = _feed(paged, (21,), decode), _feed(paged, chunks, decode)
    n = 31 + decode
    assert cut.host_lengths == whole.host_lengths == [n, 3 + decode]
    for i in range(2):
        a, b = whole.weights[i][0, :, :n], cut.weights[i][0, :, :n]
        # the sums are one row's weights (of 1 a query head) on those of the steps before
        assert (a.sum() - 4 * (1 + decode)).abs() < 1e-3 and (a > 0).all()
        # fp32 throughout: keys and queries to 1e-4 of their size, as in the prompts' own tests
        assert ((a - b).abs() <= 1e-3 * a + 1e-6).all()
        assert torch.equal(whole.weights[i][1, :, :3 + decode], cut.weights[i][1, :, :3 + decode])


def test_weights_that_were_followed_by_a_step_stay():
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=256)
    cache = _feed(paged, (20,))
    before = [w[0, :, :30].clone() for w in cache.weights]
    paged.step(torch.tensor([1, 2], device=DEV), cache)
    paged.prefill([[3], []], cache)
    for i in range(2):
        assert (cache.weights[i][0, :, :30] >= before[i]).all()
        assert (cache.weights[i][0, :, :32].sum() - 4 * 3).abs() < 1e-3  # two last tokens' and a step's
    paged.prefill([_tokens(9, 4), []], cache)
    assert cache.host_lengths[0] == 41 and not cache._provisional
    paged.step(torch.tensor([1, 2], device=DEV), cache)
    assert cache.host_lengths[0] == 25


def test_a_sequence_in_the_range_is_evicted_by_its_last_token():
    """Another one's growth evicts it before it attends again."""
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=256)
    cache = _feed(paged, (10, 10))
    weights = [w[0, :, :30].clone() for w in cache.weights]
    assert cache.host_lengths[0] == 30 and all((w > 0).all() for w in weights)
    paged.prefill([[], _tokens(40, 6)], cache)
    paged.step(torch.tensor([1, 2], device=DEV), cache, [False, True])
    assert cache.host_lengths == [24, 25]
    for i in range(2):
        for h in range(2):
            kept = set(cache.pos[i][0, h, :24].tolist())
            order = weights[i][h, 1:28].argsort(descending=True).tolist()
            assert kept == {0, 28, 29} | {1 + x for x in order[:21]}


def test_other_weights_settle_what_was_provisional():
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=256)
    cache = _feed(paged, (20,))
    q = torch.randn(2, 4, 128, device=DEV)[..., :cache.D].contiguous()
    for i in range(2):
        cache.weigh(i, q, torch.tensor([30, 0], dtype=torch.int32, device=DEV))
    paged.prefill([[3], []], cache)
    for i in range(2):  # the last token's, these and the new last token's
        assert (cache.weights[i][0, :, :31].sum() - 4 * 3).abs() < 1e-3


def test_refused_chunks_take_nothing_back():
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=256)
    cache = _feed(paged, (20,))
    before = [w.clone() for w in cache.weights]
    with pytest.raises(AssertionError):
        paged.prefill([_tokens(90, 5), []], cache)
    assert all(torch.equal(a, b) for a, b in zip(before, cache.weights)) and 0 in cache._provisional
    cache.release(0)
    assert not cache._provisional
