"""Refusals and page handling of the paged cache and decoder that need no GPU: what is refused
changes nothing, and what a sequence holds is followed everywhere."""
from __future__ import annotations

import pytest
import torch


def _decoder(rows):
    from dcr_b200.models.llama.model import DCRLlamaDecoder, LlamaDecodeConfig
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    cfg = LlamaDecodeConfig(vocab=50, hidden=128, intermediate=128, layers=1, heads=2, kv_heads=1)
    model = DCRLlamaDecoder(cfg, attention="dense", dtype=torch.float32, device="cpu", seed=0)
    return PagedLlamaDecoder(model, max_positions=rows)


def _state(c):
    return (list(c.host_lengths), list(c.host_seen), [list(p) for p in c.host_pages],
            list(c.free_pages), c.lengths.tolist(), c.seen.tolist(), c.queried.tolist(),
            c.page_table.tolist(), c._tokens)


def _refused(c, call, *args):
    before = _state(c)
    with pytest.raises(AssertionError):
        call(*args)
    assert _state(c) == before


def test_positions_past_the_table_are_refused_before_anything_changes():
    paged = _decoder(4)
    cache = paged.new_cache(3, 10, 40, page_size=8)
    _refused(cache, paged.prefill, [[1, 2, 3, 4, 5], [1], []], cache)
    cache.reserve([4, 2, 0])
    _refused(cache, paged.step, torch.tensor([1, 2, 3]), cache)
    _refused(cache, paged.step, torch.tensor([1, 2, 3]), cache, [True, False, False])


def test_a_refused_step_does_not_evict():
    paged = _decoder(4)
    cache = paged.new_cache(2, 10, 40, page_size=8, budget=3, sinks=0, recent=1)
    cache.reserve([4, 1])
    cache.evict = lambda: pytest.fail("evicted")
    _refused(cache, paged.step, torch.tensor([1, 2]), cache)
    _refused(cache, paged.step, torch.tensor([1, 2]), cache, [True])


@pytest.mark.parametrize("tokens", [torch.tensor([1, 2]), torch.tensor([[1], [2], [3]]),
                                    torch.tensor([1.0, 2.0, 3.0])])
def test_tokens_that_are_not_one_id_a_sequence_are_refused(tokens):
    paged = _decoder(64)
    cache = paged.new_cache(3, 10, 40, page_size=8)
    cache.reserve([4, 2, 1])
    _refused(cache, paged.step, tokens, cache)
    _refused(cache, paged.step, tokens, cache, [True, False, True])


def test_generate_wants_a_prompt_for_every_sequence():
    paged = _decoder(64)
    cache = paged.new_cache(2, 10, 40, page_size=8)
    for prompts in ([[1]], [[1], [2], [3]]):
        _refused(cache, paged.generate, prompts, cache, 3)


@pytest.mark.parametrize("prompt", [[50], [3, -1], [1, 2, 1 << 40]])
def test_prompt_ids_outside_the_vocabulary_are_refused(prompt):
    paged = _decoder(64)
    cache = paged.new_cache(2, 10, 40, page_size=8)
    _refused(cache, paged.prefill, [[1], prompt], cache)
    _refused(cache, paged.generate, [[1], prompt], cache, 3)


def test_eviction_and_release_reach_what_is_attended_to(monkeypatch):
    from dcr_b200 import paged_cache
    monkeypatch.setattr(paged_cache, "paged_evict", lambda *a, **kw: None)
    cache = paged_cache.PagedKVCache(2, 3, 2, 20, 40, page_size=8, dtype=torch.bfloat16, device="cpu",
                                     budget=10, sinks=1, recent=2)
    cache.reserve([30, 9, 12])
    assert cache.queried.tolist() == [30, 9, 12]
    cache.evict()
    assert cache.queried.tolist() == cache.lengths.tolist() == [10, 9, 10]
    cache.reserve([1, 0, 1])
    assert cache.queried.tolist() == [11, 0, 11]
    cache.evict()
    assert cache.queried.tolist() == [10, 0, 10]  # the second has asked for nothing since
    cache.reserve([1, 1, 1])
    cache.release(0)
    assert cache.queried.tolist() == [0, 10, 11] and cache.lengths.tolist() == [0, 10, 11]


def test_tokens_reserved_before_an_eviction_are_not_appended_after_it(monkeypatch):
    from dcr_b200 import paged_cache
    monkeypatch.setattr(paged_cache, "paged_evict", lambda *a, **kw: None)
    monkeypatch.setattr(paged_cache, "paged_append", lambda *a, **kw: a[0])
    cache = paged_cache.PagedKVCache(1, 2, 2, 20, 40, page_size=8, dtype=torch.bfloat16, device="cpu",
                                     budget=10, sinks=1, recent=2)
    cache.reserve([9, 3])
    cache.evict()                      # nothing is over the budget
    cache.append(0, 1, 2, 3, 4, 5)
    cache.reserve([4, 1])
    cache.evict()                      # slots 9 to 12 are gone
    with pytest.raises(AssertionError):
        cache.append(0, 1, 2, 3, 4, 5)
    cache.reserve([1, 1])
    cache.append(0, 1, 2, 3, 4, 5)
