"""The paged decoder on the GPU: prompts in chunks and beside running sequences, a common prefix, and
rotation from frequencies."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _model(dtype=torch.float32, layers=2, seed=0):
    from dcr_b200.models.llama.model import DCRLlamaDecoder, LlamaDecodeConfig
    cfg = LlamaDecodeConfig(vocab=512, hidden=256, intermediate=512, layers=layers, heads=4, kv_heads=2)
    return DCRLlamaDecoder(cfg, attention="dense", dtype=dtype, device=DEV, seed=seed)


def _close(a, b):
    # fp32 throughout: sums in other orders over a few hundred terms and two layers
    return (a - b).abs().max() <= 1e-4 * b.abs().max()


def _tokens(n, seed):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _alone(paged, tokens):
    """The logits after a sequence's last token, fed whole into a cache of its own."""
    return paged.prefill([tokens], paged.new_cache(1, 40, 256, page_size=8))[0]


def test_chunks_are_the_whole_prompt():
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=256)
    a, b = _tokens(100, 1), _tokens(37, 2)
    cache = paged.new_cache(2, 40, 128, page_size=8)
    paged.prefill([a[:33], b[:1]], cache)
    paged.prefill([a[33:34], []], cache)
    x = paged.prefill([a[34:], b[1:]], cache)
    assert cache.host_lengths == [100, 37]
    assert _close(x[0], _alone(paged, a)) and _close(x[1], _alone(paged, b))


def test_a_prompt_beside_running_sequences():
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=256)
    a, b, c = _tokens(20, 3), _tokens(30, 4), _tokens(50, 5)
    cache = paged.new_cache(3, 40, 64, page_size=8)
    paged.prefill([a, b, []], cache)
    a.append(7), b.append(8)
    paged.step(torch.tensor([7, 8, 0], device=DEV), cache, [True, True, False])
    x = paged.prefill([[], [], c], cache)  # the others wait
    assert _close(x[2], _alone(paged, c)) and (x[:2] == 0).all()
    y = paged.step(torch.tensor([1, 2, 3], device=DEV), cache)
    for row, s, t in zip(y, (a, b, c), (1, 2, 3)):
        assert _close(row, _alone(paged, s + [t]))


@pytest.mark.parametrize("n", [5, 16, 43])
def test_a_prefix_is_held_once(n):
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=256)
    prefix, parts = _tokens(n, 6), [_tokens(3, 7), [], _tokens(20, 8), _tokens(1, 9)]
    cache = paged.new_cache(4, 40, 128, page_size=8)
    x = paged.prefill(parts, cache, prefix=prefix)
    for row, p in zip(x, parts):
        assert _close(row, _alone(paged, prefix + p)) if p else (row == 0).all()
    used = 40 - len(cache.free_pages)
    want = n // 8 + sum(-(-(n + len(p)) // 8) - n // 8 for p in parts if p)
    assert used == want
    full = [prefix + p for p in parts]
    for t in (11, 12):
        x = paged.step(torch.tensor([t] * 4, device=DEV), cache, [True, False, True, True])
        for b in (0, 2, 3):
            full[b].append(t)
            assert _close(x[b], _alone(paged, full[b]))
    for b in (0, 2, 3):
        cache.release(b)
    assert len(cache.free_pages) == 40


def test_generate_on_a_prefix():
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(dtype=torch.float32), max_positions=256)
    prefix, parts = _tokens(30, 10), [[1, 2], [3], [4, 5, 6]]
    got = paged.generate(parts, paged.new_cache(3, 40, 128, page_size=8), 10, prefix=prefix)
    want = paged.generate([prefix + p for p in parts], paged.new_cache(3, 40, 128, page_size=8), 10)
    assert got == want  # greedy tokens: near ties would need logits equal to 1e-4 of the largest
    again = paged.generate([[1, 2]] * 3, paged.new_cache(3, 40, 128, page_size=16), 10, prefix=prefix)
    assert again[0] == again[1] == again[2] == want[0]


def test_prefix_refusals_change_nothing():
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=64)
    cache = paged.new_cache(2, 6, 40, page_size=8)
    for prompts, prefix in (([[1], [2]], [600]), ([[1], [2]], [1] * 64), ([[1] * 20, [2]], [1] * 30),
                            ([[1] * 9, [2] * 9], [1] * 31), ([[], []], [1])):
        with pytest.raises(AssertionError):
            paged.prefill(prompts, cache, prefix=prefix)
        assert cache.host_lengths == [0, 0] and len(cache.free_pages) == 6
    paged.prefill([[1], [2]], cache, prefix=[1] * 9)
    with pytest.raises(AssertionError):
        paged.prefill([[1], [2]], cache, prefix=[1])
    with pytest.raises(AssertionError):
        PagedLlamaDecoder(_model(), interleaved=True)


def test_rotation_from_frequencies():
    """The model's own frequencies give the tables' logits; an interleaved part of the head differs."""
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    model = _model()
    plain = PagedLlamaDecoder(model, max_positions=256, qk_norm=True)
    free = PagedLlamaDecoder(model, max_positions=8, qk_norm=True, inv_freq=model.inv_freq)
    part = PagedLlamaDecoder(model, max_positions=8, qk_norm=True, inv_freq=model.inv_freq[:16], interleaved=True)
    tokens = _tokens(60, 11)
    want = _alone(plain, tokens)
    assert _close(_alone(free, tokens), want)
    other = _alone(part, tokens)
    assert torch.isfinite(other).all() and not _close(other, want)
    cache = part.new_cache(1, 10, 64, page_size=8)
    part.prefill([tokens[:50]], cache)
    for t in tokens[50:]:
        x = part.step(torch.tensor([t], device=DEV), cache)
    assert _close(x[0], other)


def test_prompts_in_a_cache_with_a_budget():
    """A chunk that takes a sequence over the budget: evicted before the next step, which attends to what
    is left."""
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=256)
    cache = paged.new_cache(2, 30, 96, page_size=8, budget=32, sinks=2, recent=8)
    paged.prefill([_tokens(30, 12), _tokens(5, 13)], cache)
    assert (cache.weights[0] == 0).all()
    paged.prefill([_tokens(20, 14), []], cache)
    assert cache.host_lengths == [50, 5] and (cache.weights[0][0, :, :50] > 0).all()
    assert (cache.weights[0][1] == 0).all()
    x = paged.step(torch.tensor([1, 2], device=DEV), cache)
    assert cache.host_lengths == [33, 6] and torch.isfinite(x).all()
    paged.prefill([_tokens(3, 15), _tokens(40, 16)], cache)  # over the budget by one: evicted first
    assert cache.host_lengths == [35, 46]
