"""Decode steps over pages that sequences share, by the shared call and by the plain one: the same answers
while sequences end, wait and begin among the others."""
from __future__ import annotations

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_paged_prompts import DEV, _close, _model, _tokens  # noqa: E402

pytestmark = pytest.mark.gpu


def _calls(monkeypatch):
    """Counts the shared calls."""
    from dcr_b200 import paged_cache
    plain, calls = paged_cache.paged_shared_attention, []

    def counted(*a, **kw):
        calls.append(a[5].tolist())
        return plain(*a, **kw)
    monkeypatch.setattr(paged_cache, "paged_shared_attention", counted)
    return calls


@pytest.mark.parametrize("n", [16, 43])
def test_sequences_that_come_and_go(n, monkeypatch):
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=256)
    calls, prefix, parts = _calls(monkeypatch), _tokens(n, 1), [_tokens(1 + b, 2 + b) for b in range(6)]
    caches = [paged.new_cache(6, 90, 128, page_size=8) for _ in range(2)]
    caches[0].shared_bytes, caches[1].shared_bytes = 0, float("inf")
    for c in caches:
        paged.prefill(parts, c, prefix=prefix)

    def step(t, live):
        x, y = (paged.step(torch.tensor([t] * 6, device=DEV), c, live) for c in caches)
        rows = [b for b in range(6) if live[b]]
        assert _close(x[rows], y[rows])

    def both(f):
        for c in caches:
            f(c)
    step(7, [True] * 6)
    assert calls == [[0, 6]] * 2
    step(8, [False, True, True, False, True, True])    # the group's first one waits
    both(lambda c: c.release(2))
    step(9, [True, True, False, True, True, True])
    both(lambda c: paged.prefill([[], [], _tokens(20, 9), [], [], []], c))  # its place is taken
    step(10, [True] * 6)
    both(lambda c: c.release(0))
    both(lambda c: c.release(1))
    step(11, [False, False, True, True, True, True])
    assert calls[-1] == [0, 3, 6]
    both(lambda c: c.fork(3, [0, 1]))
    step(12, [True] * 6)
    step(13, [True, False, True, False, False, False])
    for b in range(6):
        both(lambda c: c.release(b))
        if b < 5:
            step(14 + b, [x > b for x in range(6)])
    assert len(calls) >= 2 * 10 and all(len(c.free_pages) == 90 for c in caches)


def test_generation_that_ends_sequence_by_sequence(monkeypatch):
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=256)
    prefix, parts = _tokens(30, 10), [[1 + b] for b in range(8)]
    plain = paged.generate(parts, paged.new_cache(8, 90, 128, page_size=8), 12, prefix=prefix)
    stop = max(range(512), key=lambda t: len({p.index(t) for p in plain if t in p}))
    calls = _calls(monkeypatch)
    want = paged.generate(parts, paged.new_cache(8, 90, 128, page_size=8), 12, prefix=prefix, stop=stop)
    assert not calls
    cache = paged.new_cache(8, 90, 128, page_size=8)
    cache.shared_bytes = 0
    # greedy tokens: near ties would need logits equal to 1e-4 of the largest
    assert paged.generate(parts, cache, 12, prefix=prefix, stop=stop) == want
    assert calls and len(cache.free_pages) == 90


def test_a_captured_call_reads_the_present_groups():
    """attend over the cache's own buffers, replayed after sequences grew and one was released."""
    from dcr_b200.paged_cache import PagedKVCache
    g = torch.Generator(device=DEV).manual_seed(1)
    c = PagedKVCache(1, 5, 2, 60, 96, page_size=8, D=64, dtype=torch.bfloat16, device=DEV)
    c.shared_bytes = 0
    for pool in c.k + c.v:
        pool.copy_(torch.randn(pool.shape, generator=g, device=DEV))
    c.reserve([50, 0, 0, 0, 0])
    c.fork(0, [1, 2, 3, 4])
    c.reserve([1] * 5)
    q = torch.randn(5, 8, 64, generator=g, device=DEV).bfloat16()
    c.attend(0, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = c.attend(0, q)
    for change in (lambda: c.reserve([1, 2, 1, 9, 1]), lambda: c.release(2), lambda: c.reserve([1, 1, 0, 0, 1])):
        change()
        graph.replay()
        assert torch.equal(o, c.attend(0, q)) and torch.isfinite(o).all()
    assert c.groups.tolist() == [0, 5] and (o[[2, 3]] == 0).all() and (o[[0, 1, 4]] != 0).any(-1).all()
