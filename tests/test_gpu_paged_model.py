"""The paged decoder on the GPU: the same logits as the model over contiguous caches, query/key
norms, ragged prompts, eviction in the loop and processed logits."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _model(dtype=torch.float32, layers=2, seed=0):
    from dcr_b200.models.llama.model import DCRLlamaDecoder, LlamaDecodeConfig
    cfg = LlamaDecodeConfig(vocab=512, hidden=256, intermediate=512, layers=layers, heads=4, kv_heads=2)
    return DCRLlamaDecoder(cfg, attention="dense", dtype=dtype, device=DEV, seed=seed)


def _dense_logits(model, sequence):
    """The logits after each token of one sequence, by the model over contiguous caches."""
    caches = model.new_caches(1, len(sequence))
    cos, sin = model.rope_table(len(sequence))
    return torch.cat([model.step(torch.tensor([t], device=DEV), caches, cos[i:i + 1], sin[i:i + 1])
                      for i, t in enumerate(sequence)])


def test_ragged_prompts_and_steps_match_contiguous_caches():
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    model = _model()
    paged = PagedLlamaDecoder(model, max_positions=64)
    g = torch.Generator().manual_seed(1)
    seqs = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (30, 9, 17)]
    cache = paged.new_cache(3, 20, 64, page_size=8)
    got = [[], [], []]
    logits = paged.prefill([s[:len(s) - 6] for s in seqs], cache)
    for i in range(6, -1, -1):
        for b in range(3):
            got[b].append(logits[b])
        if i:
            logits = paged.step(torch.tensor([s[len(s) - i] for s in seqs], device=DEV), cache)
    assert cache.host_lengths == [30, 9, 17]
    for b, s in enumerate(seqs):
        want = _dense_logits(model, s)[-7:]
        # fp32 throughout: sums in other orders over a few hundred terms and two layers
        assert (torch.stack(got[b]) - want).abs().max() <= 1e-4 * want.abs().max()


def test_idle_sequences_keep_their_state():
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=64)
    prompts = [[1, 2, 3, 4], [5, 6, 7, 8, 9], [10, 11]]
    one = paged.new_cache(3, 20, 40, page_size=8, budget=20, sinks=1, recent=2)
    two = paged.new_cache(3, 20, 40, page_size=8, budget=20, sinks=1, recent=2)
    paged.prefill(prompts, one), paged.prefill(prompts, two)
    tokens = torch.tensor([20, 21, 22], device=DEV)
    a = paged.step(tokens, one)
    b = paged.step(tokens, two, [True, False, True])
    assert (a[[0, 2]] - b[[0, 2]]).abs().max() <= 1e-5 and two.host_lengths == [5, 5, 3]
    assert (two.weights[0][1] == 0).all() and (two.weights[0][0, :, :5] > 0).all()
    c = paged.step(tokens, two, [False, True, False])
    assert (a[1] - c[1]).abs().max() <= 1e-5
    assert torch.allclose(one.weights[1][..., :6], two.weights[1][..., :6], atol=1e-5)


def test_query_and_key_norms():
    """One layer's attention against torch: norms of the heads, rotation, attention."""
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    model = _model(layers=1)
    paged = PagedLlamaDecoder(model, qk_norm=True, max_positions=64)
    g = torch.Generator(device=DEV).manual_seed(3)
    with torch.no_grad():
        paged.q_norm[0].copy_(torch.randn(64, generator=g, device=DEV))
        paged.k_norm[0].copy_(torch.randn(64, generator=g, device=DEV))
    prompt = [3, 1, 4, 1, 5, 9, 2, 6]
    cache = paged.new_cache(1, 4, 32, page_size=8)
    paged.prefill([prompt[:-1]], cache)
    logits = paged.step(torch.tensor(prompt[-1:], device=DEV), cache)
    layer, cfg = model.layers[0], model.cfg
    x = model.embed_tokens(torch.tensor(prompt, device=DEV)).double()
    rms = lambda t, w, eps: t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * w.double()  # noqa: E731
    h = rms(x, layer.input_layernorm.weight, 1e-5)
    q = (h @ layer.self_attn.q_proj.weight.double().T).view(8, 4, 64)
    k = (h @ layer.self_attn.k_proj.weight.double().T).view(8, 2, 64)
    v = (h @ layer.self_attn.v_proj.weight.double().T).view(8, 2, 64)
    cos, sin = (t.double()[:, None] for t in model.rope_table(8))
    turn = lambda t: t * cos + torch.cat((-t[..., 32:], t[..., :32]), -1) * sin  # noqa: E731
    q, k = turn(rms(q, paged.q_norm[0], 1e-5)), turn(rms(k, paged.k_norm[0], 1e-5))
    k, v = k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)
    p = torch.softmax(torch.einsum("hd,nhd->hn", q[-1], k) / 8, -1)
    o = torch.einsum("hn,nhd->hd", p, v).reshape(1, -1)
    y = x[-1:] + o @ layer.self_attn.o_proj.weight.double().T
    z = rms(y, layer.post_attention_layernorm.weight, 1e-5)
    gate, up = z @ layer.gate_proj.weight.double().T, z @ layer.up_proj.weight.double().T
    y = y + (gate / (1 + torch.exp(-gate)) * up) @ layer.down_proj.weight.double().T
    want = rms(y, model.norm.weight, 1e-5) @ model.embed_tokens.weight.double().T
    assert (logits.double() - want).abs().max() <= 1e-4 * want.abs().max()


@pytest.mark.parametrize("slack", [1, 5])
def test_eviction_in_the_loop(slack):
    """Every step attends to exactly the slots that are left, and these obey the budget."""
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=128)
    cache = paged.new_cache(2, 12, 40, page_size=8, budget=24, sinks=2, recent=6, slack=slack)
    g = torch.Generator().manual_seed(5)
    paged.prefill([torch.randint(0, 512, (n,), generator=g).tolist() for n in (24, 10)], cache)
    seen_q = {}
    plain = cache.attend

    def attend(i, q, **kw):
        o = plain(i, q, **kw)
        for b in range(2):  # over the rows the cache holds for this sequence, in any order
            K, V = (t.double() for t in cache.gather(i, b))
            z = torch.einsum("hd,hnd->hn", q[b].double(), K.repeat_interleave(2, 0)) / 8
            want = torch.einsum("hn,hnd->hd", torch.softmax(z, -1), V.repeat_interleave(2, 0))
            assert (o[b].double() - want).abs().max() <= 1e-5
        seen_q[i] = q
        return o

    cache.attend = attend
    for step in range(40):
        paged.step(torch.randint(0, 512, (2,), generator=g).to(DEV), cache)
        for b, n in enumerate(cache.host_lengths):
            assert n <= 24 + slack
            for i in range(2):
                for h in range(2):
                    pos = sorted(cache.pos[i][b, h, :n].tolist())
                    assert len(set(pos)) == n and pos[:2] == [0, 1]
                    last = cache.host_seen[b]
                    assert pos[-min(6, n):] == list(range(last - min(6, n), last))
    assert cache.host_seen == [64, 50] and sum(map(len, cache.host_pages)) + len(cache.free_pages) == 12
    assert set(seen_q) == {0, 1}


def test_generate_with_penalties_masks_and_stops():
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    model = _model(dtype=torch.bfloat16)
    paged = PagedLlamaDecoder(model, qk_norm=True, max_positions=128)
    prompts = [[7, 8, 9], [100, 101], [3] * 20]
    greedy = paged.generate(prompts, paged.new_cache(3, 40, 64, page_size=8), 12)
    assert [len(t) for t in greedy] == [12, 12, 12]
    again = paged.generate(prompts, paged.new_cache(3, 40, 64, page_size=16), 12)
    assert again == greedy  # other pages, the same tokens
    # a penalty no token survives a second time
    once = paged.generate(prompts, paged.new_cache(3, 40, 64, page_size=8), 12,
                          frequency=torch.full((3,), 1e4, device=DEV))
    assert all(len(set(t)) == 12 for t in once)
    # a grammar that allows tokens 32..39 only, and nothing after four of them for sequence 1
    def grammar(out):
        words = torch.zeros(3, 16, dtype=torch.int32)
        words[:, 1] = 0xff
        if len(out[1]) == 4:
            words[1] = 0
        return words.to(DEV)
    cache = paged.new_cache(3, 40, 64, page_size=8, budget=16, sinks=1, recent=4)
    told = paged.generate(prompts, cache, 12, allowed=grammar)
    assert [len(t) for t in told] == [12, 4, 12] and all(32 <= x < 40 for t in told for x in t)
    assert len(cache.free_pages) == 40
    stop = greedy[0][2]
    ended = paged.generate(prompts, paged.new_cache(3, 40, 64, page_size=8), 12, stop=stop)
    assert ended[0] == greedy[0][:greedy[0].index(stop) + 1]
    assert math.isfinite(sum(map(len, ended)))
