"""Pages that sequences share (CPU): forks, what they hold, and when pages come back."""
from __future__ import annotations

import pytest
import torch


def _cache(**kw):
    from dcr_b200.paged_cache import PagedKVCache
    return PagedKVCache(**{**dict(layers=2, batch=4, H_kv=2, pages=12, max_slots=40, page_size=8,
                                  dtype=torch.float32, device="cpu"), **kw})


def _check(c, pages=12):
    """Every page is free or held, as often as it is counted."""
    held = [p for pages in c.host_pages for p in pages]
    assert sorted(set(held) | set(c.free_pages)) == list(range(pages))
    assert not set(held) & set(c.free_pages)
    assert all(c._holders[p] == held.count(p) for p in range(pages))
    for b, n in enumerate(c.host_lengths):
        m = -(-n // c.page_size)
        assert c.page_table[b].tolist() == c.host_pages[b] + [-1] * (c.max_pages - m)
    if max(c._holders) < 2:
        assert c.groups is None
    else:
        assert (c.groups.tolist(), c.prefix.tolist()) == tuple(c.shared_groups())


def test_fork_shares_full_pages_and_copies_the_last():
    c = _cache()
    c.reserve([0, 21, 0, 0])
    for pool in c.k + c.v:
        pool.copy_(torch.randn(pool.shape))
    c.fork(1, [2, 3])
    _check(c)
    assert c.host_lengths == [0, 21, 21, 21] and c.host_seen == [0, 21, 21, 21]
    assert c.host_pages[2][:2] == c.host_pages[1][:2] == c.host_pages[3][:2]
    assert len({c.host_pages[b][2] for b in (1, 2, 3)}) == 3 and len(c.free_pages) == 12 - 5
    for layer in range(2):
        want = c.gather(layer, 1)
        for b in (2, 3):
            assert all(torch.equal(x, y) for x, y in zip(c.gather(layer, b), want))
    assert c.groups.tolist() == [0, 1, 4] and c.prefix.tolist() == [0, 16, 16, 16]
    c.reserve([0, 0, 5, 0])  # grows into a page of its own
    _check(c)
    assert c.host_pages[2][:2] == c.host_pages[1][:2] and c.starts.tolist() == [0, 0, 0, 5, 5]
    c.release(1)
    _check(c)
    assert c.groups.tolist() == [0, 1, 2, 4] and c.prefix.tolist() == [0, 0, 16, 16]
    c.release(2), c.release(3)
    _check(c)
    assert len(c.free_pages) == 12 and c.groups is None


def test_fork_of_full_pages_needs_no_page():
    c = _cache(pages=2)
    c.reserve([16, 0, 0, 0])
    c.fork(0, [1, 2, 3])
    _check(c, 2)
    assert not c.free_pages and c.prefix.tolist() == [16] * 4
    with pytest.raises(AssertionError):
        c.reserve([1, 0, 0, 0])
    for b in (0, 1, 2):
        c.release(b)
        assert not c.free_pages
    c.release(3)
    assert len(c.free_pages) == 2


def test_fork_of_a_fork_and_groups_apart():
    c = _cache()
    c.reserve([20, 0, 9, 0])
    c.fork(0, [1])
    c.fork(2, [3])
    _check(c)
    assert c.groups.tolist() == [0, 2, 4] and c.prefix.tolist() == [16, 16, 8, 8]
    c.release(0)
    c.fork(1, [0])
    _check(c)
    assert c.prefix.tolist() == [16, 16, 8, 8]


def test_fork_refusals_change_nothing():
    c = _cache()
    c.reserve([20, 0, 5, 0])
    before = ([list(p) for p in c.host_pages], list(c.free_pages), list(c._holders), list(c.host_lengths))
    for b, others in ((1, [3]), (0, [0]), (0, [2]), (0, [1, 1]), (0, [4]), (9, [1]), (-1, [1])):
        with pytest.raises(AssertionError):
            c.fork(b, others)
    small = _cache(pages=3)
    small.reserve([20, 0, 0, 0])
    with pytest.raises(AssertionError):
        small.fork(0, [1])
    with pytest.raises(AssertionError):
        budget = _cache(budget=16, sinks=1, recent=2)
        budget.reserve([9, 0, 0, 0])
        budget.fork(0, [1])
    assert before == (c.host_pages, c.free_pages, c._holders, c.host_lengths)


def test_eviction_counts_pages():
    c = _cache(budget=16, sinks=1, recent=2)
    c.reserve([30, 0, 0, 0])
    c._resize(0, 16)
    c._publish([0])
    _check(c)


def test_attention_before_tokens_is_refused():
    c = _cache()
    x = torch.zeros(1, 2, 64)
    with pytest.raises(AssertionError):
        c.prefill_attend(0, x)
    with pytest.raises(AssertionError):
        c.append_rotary(0, x, x, x, torch.ones(32))
