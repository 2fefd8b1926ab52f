"""The paged cache's page handling (CPU): pages follow lengths, run out, come back."""
from __future__ import annotations

import pytest
import torch


def _cache(**kw):
    from dcr_b200.paged_cache import PagedKVCache
    return PagedKVCache(**{**dict(layers=2, batch=3, H_kv=2, pages=10, max_slots=40, page_size=8,
                                  dtype=torch.bfloat16, device="cpu"), **kw})


def _check(c):
    held = [p for pages in c.host_pages for p in pages]
    assert sorted(held + c.free_pages) == list(range(10))
    for b, n in enumerate(c.host_lengths):
        m = -(-n // c.page_size)
        assert len(c.host_pages[b]) == m
        assert c.page_table[b].tolist() == c.host_pages[b] + [-1] * (c.max_pages - m)
    assert c.lengths.tolist() == c.host_lengths and c.seen.tolist() == c.host_seen


def test_reserve_and_release():
    c = _cache()
    assert c.reserve([9, 0, 8]) == 17
    _check(c)
    seq, slots, positions = c._tokens
    assert seq.tolist() == [0] * 9 + [2] * 8 and slots.tolist() == list(range(9)) + list(range(8))
    assert torch.equal(slots, positions)
    c.reserve([1, 1, 1])
    _check(c)
    assert c._tokens[1].tolist() == [9, 0, 8] and c.host_lengths == [10, 1, 9]
    c.release(0)
    _check(c)
    assert c.host_lengths == [0, 1, 9]
    assert c.reserve([0, 0, 0]) == 0
    _check(c)


def test_refusals_change_nothing():
    c = _cache()
    c.reserve([30, 0, 0])
    for bad in ([11, 0, 0], [0, 40, 40], [1, 1], [-1, 0, 0]):
        before = (list(c.host_lengths), [list(p) for p in c.host_pages], list(c.free_pages))
        with pytest.raises(AssertionError):
            c.reserve(bad)
        assert before == (c.host_lengths, c.host_pages, c.free_pages)
    _check(c)


def test_budget_arguments():
    c = _cache(budget=16, sinks=2, recent=4, slack=4)
    c.reserve([19, 1, 0])
    assert not c.over_budget()
    c.reserve([1, 0, 0])
    assert c.over_budget()
    for kw in (dict(budget=0), dict(budget=40), dict(budget=8, sinks=4, recent=5),
               dict(budget=36, slack=5), dict(budget=8, slack=0, sinks=0, recent=0), dict(pages=0),
               dict(D=32), dict(dtype=torch.float64)):
        with pytest.raises(AssertionError):
            _cache(**kw)
    with pytest.raises(AssertionError):
        _cache().evict()
