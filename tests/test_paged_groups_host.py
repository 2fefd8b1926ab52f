"""Groups of sequences that share pages (CPU): they outlive the sequences that end, wait or begin
among them."""
from __future__ import annotations

import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_paged_prompts_host import _cache, _check  # noqa: E402


def _forked(batch, slots=32, **kw):
    c = _cache(**{**dict(batch=batch, pages=200, max_slots=64), **kw})
    c.reserve([slots] + [0] * (batch - 1))
    c.fork(0, list(range(1, batch)))
    return c


def _same(c, groups, prefix):
    _check(c, 200)
    assert c.groups.tolist() == groups and c.prefix.tolist() == prefix


def test_sequences_that_end_do_not_part_the_others():
    c = _forked(5)
    _same(c, [0, 5], [32] * 5)
    c.release(1), c.release(3)
    _same(c, [0, 5], [32, 0, 32, 0, 32])
    c.release(4)
    _same(c, [0, 5], [32, 0, 32, 0, 0])
    c.release(0)  # the last holder shares with nobody
    _check_none(c)


def _check_none(c):
    assert c.groups is None and c.prefix is None


@pytest.mark.parametrize("gone", [(10, 20, 30), (1, 2, 3), (62, 63), (5, 60)])
def test_a_batch_stays_one_group(gone):
    c = _forked(64)
    for b in gone:
        c.release(b)
    _same(c, [0, 64], [0 if b in gone else 32 for b in range(64)])


def test_a_group_that_lost_its_first():
    c = _forked(6)
    c.release(0), c.release(3)
    _same(c, [0, 1, 6], [0, 32, 32, 0, 32, 32])


def test_a_prompt_of_its_own_in_the_place_of_one_that_ended():
    c = _forked(5)
    c.release(2)
    c.reserve([1, 1, 20, 1, 1])
    _same(c, [0, 5], [32, 32, 0, 32, 32])
    c.reserve([9, 0, 1, 0, 9])
    _same(c, [0, 5], [32, 32, 0, 32, 32])
    c.fork(0, [])
    _same(c, [0, 5], [32, 32, 0, 32, 32])


def test_two_prefixes_side_by_side():
    c = _cache(batch=7, pages=200, max_slots=64)
    c.reserve([0, 32, 0, 0, 24, 0, 0])
    c.fork(1, [2, 3])
    c.fork(4, [5, 6])
    _same(c, [0, 1, 4, 7], [0, 32, 32, 32, 24, 24, 24])
    c.release(2), c.release(5)
    _same(c, [0, 1, 4, 7], [0, 32, 0, 32, 24, 0, 24])
    c.release(4)  # the second group's last holder is alone
    _same(c, [0, 1, 7], [0, 32, 0, 32, 0, 0, 0])


def test_holders_that_are_no_neighbours():
    c = _cache(batch=4, pages=200, max_slots=64)
    c.reserve([16, 16, 0, 0])
    c.fork(0, [2])
    c.fork(1, [3])  # 0 and 2, 1 and 3
    assert max(c._holders) == 2
    _check_none(c)
    c.release(1)
    _same(c, [0, 4], [16, 0, 16, 0])


def test_an_idle_sequence_among_prompts_on_a_prefix(monkeypatch):
    import torch
    from dcr_b200.models.llama import paged as module
    from test_paged_edges_host import _decoder
    decoder = _decoder(100)
    cache = decoder.new_cache(4, 200, 64, page_size=8)
    monkeypatch.setattr(module.PagedLlamaDecoder, "_layers",
                        lambda self, tokens, cache, attend: torch.zeros(tokens.shape[0], 128))
    decoder.prefill([[1], [], [2, 3], [4]], cache, prefix=[5] * 17)
    _same(cache, [0, 4], [16, 0, 16, 16])
    decoder.prefill([[], [6] * 9, [], []], cache)
    _same(cache, [0, 4], [16, 0, 16, 16])


def _moments(c, steps, monkeypatch):
    """Grows every sequence, and fails where that looks for shared pages or walks the pool."""
    class Unwalked(list):
        def __iter__(self):
            raise AssertionError("every page of the pool is looked at")
    c._holders = Unwalked(c._holders)
    with monkeypatch.context() as m:
        m.setattr(c, "shared_groups", lambda: pytest.fail("shared pages are looked for"))
        for _ in range(steps):
            c.reserve([1] * c.batch)
    c._holders = list.copy(c._holders)


def test_sequences_that_grow_look_for_no_shared_pages(monkeypatch):
    c = _forked(8)
    _moments(c, 20, monkeypatch)
    _same(c, [0, 8], [32] * 8)
    c.release(3)
    c.reserve([0, 0, 0, 9, 0, 0, 0, 0])
    _moments(c, 9, monkeypatch)
    _same(c, [0, 8], [0 if b == 3 else 32 for b in range(8)])


def test_a_cache_that_shares_nothing_looks_for_nothing(monkeypatch):
    c = _cache(batch=4, pages=200, max_slots=64)
    _moments(c, 20, monkeypatch)
    with monkeypatch.context() as m:
        m.setattr(c, "shared_groups", lambda: pytest.fail("shared pages are looked for"))
        c.release(1)
    _check_none(c)


def test_prefixes_of_any_length():
    """Forks of forks that parted at several places."""
    for slots in (1, 7, 8, 9, 16, 63, 64):
        c = _forked(4, slots)
        n = slots // 8 * 8
        if n == 0:
            _check_none(c)
            continue
        _same(c, [0, 4], [n] * 4)
    c = _cache(batch=6, pages=200, max_slots=160)
    c.reserve([8, 0, 0, 0, 0, 0])
    for b in range(1, 6):  # each goes on behind the one before it
        c.fork(b - 1, [b])
        c.reserve([0] * b + [16] + [0] * (5 - b))
    _same(c, [0, 6], [8] * 6)
    c.release(0)
    _same(c, [0, 1, 6], [0, 24, 24, 24, 24, 24])
    assert c._shared == len({p for p in range(200) if c._holders[p] > 1})


def test_what_kernels_read_stays_where_it_is():
    """Starts, groups and prefixes are written in place, as lengths are, so that a captured call reads the
    present ones."""
    c = _forked(5)
    starts, groups, prefix = c.starts, c.groups, c.prefix
    for new in ([1] * 5, [1] * 5, [0, 3, 1, 0, 1], [1] * 5, [0] * 5):
        c.reserve(new)
        assert c.starts is starts and starts.tolist() == [sum(new[:b]) for b in range(6)]
    c.release(2)
    assert c.groups.data_ptr() == groups.data_ptr() and c.prefix is prefix
    _same(c, [0, 5], [32, 32, 0, 32, 32])
    for b in (0, 1, 3):
        c.release(b)
    _check_none(c)
    c.fork(4, [0, 1, 2])
    assert c.groups.data_ptr() == groups.data_ptr() and c.prefix is prefix
    _same(c, [0, 5], [32, 32, 32, 0, 32])


def test_starts_are_copied_when_they_change_only():
    c = _cache(batch=3, pages=200, max_slots=64)
    c.reserve([1, 1, 1])
    starts = c.starts
    starts.fill_(-7)
    c.reserve([1, 1, 1])
    assert c.starts is starts and (starts == -7).all()
    c.reserve([1, 0, 1])
    assert starts.tolist() == [0, 1, 1, 2]


def test_a_step_copies_the_entries_of_its_new_pages():
    """Whatever comes and goes, the page table follows; what did not change in it is not copied."""
    import random
    rng = random.Random(5)
    c = _cache(batch=5, pages=200, max_slots=320)
    c.reserve([300, 0, 0, 0, 0])
    c.fork(0, [3])
    c.page_table[0, :37].fill_(-9)  # a step's new page is entry 38
    c.reserve([8, 0, 0, 0, 0])
    assert (c.page_table[0, :37] == -9).all() and c.page_table[0, 38] == c.host_pages[0][38]
    c.release(0)
    for _ in range(60):
        b, others = rng.randrange(5), [o for o in range(5) if c.host_lengths[o] == 0]
        if c.host_lengths[b] and rng.random() < 0.4:
            c.release(b)
        elif c.host_lengths[b] and rng.random() < 0.5:
            c.fork(b, others)
        else:
            c.reserve([min(rng.randrange(20), 320 - n) if rng.random() < 0.6 else 0 for n in c.host_lengths])
        if c.groups is not None or max(c._holders) < 2:
            _check(c, 200)
        for s in range(5):
            assert c.page_table[s].tolist() == c.host_pages[s] + [-1] * (40 - len(c.host_pages[s]))


def test_evicted_pages_leave_the_table():
    c = _cache(batch=2, pages=200, max_slots=64, budget=16, sinks=1, recent=2)
    c.reserve([60, 20])
    changed = [b for b in range(2) if c._resize(b, 16)]
    c._resize(0, 30)  # other pages in the places of those that left
    c._publish(changed)
    for s in range(2):
        assert c.page_table[s].tolist() == c.host_pages[s] + [-1] * (8 - len(c.host_pages[s]))


@pytest.mark.parametrize("gone,spans", [((0,), [0, 1, 64]), (tuple(range(40)), [0, 40, 64]), ((63,), [0, 64]),
                                        ((), [0, 64])])
def test_sequences_before_the_first_that_shares_are_one_span(gone, spans, monkeypatch):
    """A batch whose first sequences ended is two groups in a call, not one for each of them."""
    import torch
    from dcr_b200 import paged_cache
    got = []
    monkeypatch.setattr(paged_cache, "paged_shared_attention", lambda *a, **kw: got.append(a))
    c = _forked(64)
    c.shared_bytes = 0
    for b in gone:
        c.release(b)
    c.attend(0, torch.zeros(64, 2, 64))
    groups, prefix = got[0][5], got[0][6]
    assert groups.tolist() == spans and prefix.tolist() == [0 if b in gone else 32 for b in range(64)]


def test_spans_of_several_prefixes(monkeypatch):
    import torch
    from dcr_b200 import paged_cache
    got = []
    monkeypatch.setattr(paged_cache, "paged_shared_attention", lambda *a, **kw: got.append(a[5].tolist()))
    c = _cache(batch=9, pages=200, max_slots=64)
    c.shared_bytes = 0
    c.reserve([9, 0, 32, 0, 16, 0, 0, 24, 0])
    c.fork(2, [3])
    c.fork(4, [6])  # 5 waits
    c.fork(7, [8])
    c.attend(0, torch.zeros(9, 2, 64))
    c.release(4)  # 6 shares with nobody
    c.attend(0, torch.zeros(9, 2, 64))
    assert got == [[0, 2, 4, 7, 9], [0, 2, 7, 9]]


def test_the_shared_call_is_taken_where_it_saves_enough(monkeypatch):
    """2 KV heads of 64 in fp32: 1024 bytes a slot; 32 shared slots of each sequence but one."""
    import torch
    from dcr_b200 import paged_cache
    got = []
    monkeypatch.setattr(paged_cache, "paged_shared_attention", lambda *a, **kw: got.append("shared"))
    monkeypatch.setattr(paged_cache, "paged_attention", lambda *a, **kw: got.append("plain"))
    c, q = _forked(9), torch.zeros(9, 2, 64)

    def call(window=0):
        c.attend(0, q, window=window)
        return got.pop()
    assert c.shared_bytes == 1e9 and _cache(dtype=torch.float16).shared_bytes == 2e8
    c.reserve([1] * 9)
    assert call() == "plain"
    c.shared_bytes = 8 * 32 * 1024
    assert call() == "shared"
    assert call(33) == "shared" and call(32) == "plain" and call(1) == "plain" and call(1000) == "shared"
    c.reserve([1] * 8 + [0])           # the last one waits
    assert call() == "plain"
    c.shared_bytes = 7 * 32 * 1024
    assert call() == "shared" and call(34) == "shared" and call(33) == "plain"
    c.reserve([0] + [1] * 8)           # the first one does
    assert call() == "shared"
    c.release(0)
    assert call() == "shared"
    c.release(4)
    assert call() == "plain"
    c.shared_bytes = 6 * 32 * 1024
    assert call() == "shared"
    for b in (1, 2, 3, 5, 6, 7):
        c.release(b)
    assert c.groups is None and call() == "plain"
