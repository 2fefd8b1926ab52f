"""The paged serving operators on the GPU where they can go wrong by their surroundings: weights far
below a row's largest, flags, table entries that no slot uses, pages that are not mapped."""
from __future__ import annotations

import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _status():
    from dcr_b200 import _lib
    return _lib.read_device_status(clear=True)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [4, 16])
@pytest.mark.parametrize("nats", [14.5, 16.0, 18.0, 20.0])
def test_f16_weights_far_below_the_largest(D, G, nats):
    """One slot far ahead of all others with a value row of zeros: O is the others' alone. The
    sequences share their pages, and are so many that a warp walks whole rows."""
    from dcr_b200.kernel.cuda.paged import paged_attention
    n, page, B, H_kv = 8192, 64, 320, 8
    pages = n // page
    k = torch.zeros(pages, H_kv, page, D, dtype=torch.float16, device=DEV)
    k[0, :, 3, 0] = nats
    v = (0.5 + torch.rand(pages, H_kv, page, D, generator=_gen(1), device=DEV)).half()
    v[0, :, 3] = 0
    q = torch.zeros(B, G * H_kv, D, dtype=torch.float16, device=DEV)
    q[:, :, 0] = 1
    table = torch.arange(pages, dtype=torch.int32, device=DEV).expand(B, pages).contiguous()
    o, lse = paged_attention(q, k, v, table, _i32([n] * B), scale=1.0, return_lse=True)
    assert _status() == 0
    # every row's maximum is nats, so all its weights are against e^nats
    rest = v.double().sum((0, 2)) * math.exp(-nats)                  # [H_kv, D]
    total = 1 + (n - 1) * math.exp(-nats)
    want = (rest / total).repeat_interleave(G, 0)
    # A weight enters in two fp16 parts on a scale where the row's largest is 2^7 at least: off by
    # 2^-22 of itself or, among the subnormals, by 2^-25 of that scale, so 2^-32 of the largest. fp32
    # sums of n terms; one rounding to fp16 (subnormal steps of 2^-24).
    part = want.abs()
    tol = n * 2.0 ** -32 * v.double().max() / total + part * (2.0 ** -21 + (n + 64) * 2 * ref.EPS)
    tol = tol + 2.0 ** -11 * (want.abs() + tol) + 2.0 ** -25
    off = ((o.double() - want).abs() / tol).max()
    assert off <= 1, (float(off), float(((o.double() - want).abs() / want).max()))
    # the denominators: fp32 sums of n terms, whatever their order
    lse_tol = (n + 64) * 2 * ref.EPS + 64 * ref.EPS * nats
    assert (lse.double() - (nats + math.log(total))).abs().max() <= lse_tol


def test_return_lse_takes_any_truth_value():
    from dcr_b200.kernel.cuda.paged import paged_attention
    k, v, table = ref.make_pool([40], 2, 16, 64, torch.bfloat16, DEV, _gen(2))
    q = torch.randn(1, 4, 64, generator=_gen(3), device=DEV).to(torch.bfloat16)
    o, lse = paged_attention(q, k, v, table, _i32([40]), return_lse=True)
    got = paged_attention(q, k, v, table, _i32([40]), return_lse=1)
    assert isinstance(got, tuple) and torch.equal(got[0], o) and torch.equal(got[1], lse)
    for no in (0, False, None):
        assert torch.equal(paged_attention(q, k, v, table, _i32([40]), return_lse=no), o)


def _evicted(lengths, budget, spoil, width=None, page=16):
    """(k, v before; k, v after; table, weights, pos, results) of one eviction; `spoil` changes the
    page table after the pool is filled."""
    from dcr_b200.kernel.cuda.paged import paged_evict
    g = _gen(budget)
    k, v, table = ref.make_pool(lengths, 2, page, 64, torch.bfloat16, DEV, g, width=width, garbage=0.0)
    cap = table.shape[1] * page
    w = torch.rand(len(lengths), 2, cap, generator=g, device=DEV)
    pos = torch.arange(cap, dtype=torch.int32, device=DEV).expand(len(lengths), 2, cap).contiguous()
    spoil(table, k.shape[0])
    k0, v0 = k.clone(), v.clone()
    assert _status() == 0
    out = paged_evict(k, v, table, _i32(lengths), w, pos, _i32([cap] * len(lengths)), budget)
    return k0, v0, k, v, table, w, pos, out


def _plan(w, lengths, budget, b, h):
    n = lengths[b]
    return ref.evict(w[b, h, :n].tolist(), list(range(n)), n, 1 << 20, budget, 0, 0)


@pytest.mark.parametrize("lengths", [[100, 20, 0], [42, 41, 40], [40, 3, 0]])
def test_evict_does_not_look_at_entries_past_the_length(lengths):
    def spoil(table, pages):
        for b, n in enumerate(lengths):
            table[b, -(-n // 16):] = pages + 5 + b
    k0, v0, k, v, table, w, pos, (src, wo, po, no) = _evicted(lengths, 40, spoil, width=9)
    assert _status() == 0
    for b in range(3):
        for h in range(2):
            assert src[b, h].tolist() == _plan(w, lengths, 40, b, h)


@pytest.mark.parametrize("n", [42, 100])  # few evictions, and many
@pytest.mark.parametrize("gone", [0, -1])  # a page of holes, a page of movers
def test_evict_reports_rows_without_a_page(n, gone):
    """A kept row that cannot be moved is not passed off as moved: src -1, weight 0, position -1."""
    from dcr_b200 import _lib
    budget, page = 40, 16

    def spoil(table, pages):
        table[0, gone] = -1
    k0, v0, k, v, table, w, pos, (src, wo, po, no) = _evicted([n, n], budget, spoil)
    lost = 0
    for b in range(2):
        for h in range(2):
            want = _plan(w, [n, n], budget, b, h)
            ek, ev = k0.clone(), v0.clone()
            for i, s in enumerate(want):
                fp, tp = int(table[b, s // page]), int(table[b, i // page])
                if s != i and (fp < 0 or tp < 0):
                    lost += 1
                    assert (int(src[b, h, i]), float(wo[b, h, i]), int(po[b, h, i])) == (-1, 0.0, -1)
                    continue
                assert int(src[b, h, i]) == s and float(wo[b, h, i]) == float(w[b, h, s])
                assert int(po[b, h, i]) == s
                if s != i:
                    ek[tp, h, i % page], ev[tp, h, i % page] = k0[fp, h, s % page], v0[fp, h, s % page]
            held = [int(x) for x in table[b] if x >= 0]
            assert torch.equal(k[held, h], ek[held, h]) and torch.equal(v[held, h], ev[held, h])
    assert _status() == (_lib.DCR_ERR_DEVICE_INDEX if lost else 0)


def _shared_rows(dtype=torch.float32, slots=48):
    """Per-slot tables [2, 2, slots] whose rows share elements: expanded over heads, over sequences,
    rows that begin inside one another."""
    yield torch.zeros(2, 1, slots, dtype=dtype, device=DEV).expand(2, 2, slots)
    yield torch.zeros(1, 2, slots, dtype=dtype, device=DEV).expand(2, 2, slots)
    yield torch.zeros(4 * slots, dtype=dtype, device=DEV).as_strided((2, 2, slots), (2 * slots, slots // 2, 1))


def _small(seed=2):
    k, v, table = ref.make_pool([40, 40], 2, 16, 64, torch.bfloat16, DEV, _gen(seed), garbage=0.0)
    q = torch.randn(2, 4, 64, generator=_gen(seed + 1), device=DEV).to(torch.bfloat16)
    return k, v, table, q, _i32([40, 40])


def test_written_tables_must_not_share_elements():
    from dcr_b200.kernel.cuda.paged import paged_append, paged_attention, paged_evict
    k, v, table, q, n = _small()
    cos = torch.ones(64, 64, dtype=torch.bfloat16, device=DEV)
    good, ids = torch.zeros(2, 2, 48, device=DEV), torch.zeros(2, 2, 48, dtype=torch.int32, device=DEV)
    append = lambda **kw: paged_append(q, q[:, :2], q[:, 2:], cos, cos, _i32([1, 1]), k, v, table,  # noqa: E731
                                       _i32([7, 7]), **kw)
    for w, pos in zip(_shared_rows(), _shared_rows(torch.int32)):
        for call in (lambda: paged_attention(q, k, v, table, n, weights=w), lambda: append(weights=w),
                     lambda: append(pos=pos),
                     lambda: paged_evict(k, v, table, n, good, ids, n, 30, weights_out=w),
                     lambda: paged_evict(k, v, table, n, good, ids, n, 30, pos_out=pos)):
            with pytest.raises(AssertionError, match="share"):
                call()
        # what is only read may be shared
        src, wo, po, _ = paged_evict(k.clone(), v.clone(), table, n, w, pos, n, 30)
        assert (src == torch.arange(30, device=DEV)).all() and (wo == 0).all() and (po == 0).all()
    plain = torch.zeros(2, 2, 48, device=DEV)
    paged_attention(q, k, v, table, n, weights=plain)
    for apart in (torch.zeros(2, 2, 48, device=DEV).transpose(0, 1), torch.zeros(2, 4, 50, device=DEV)[:, ::2, 1:49],
                  torch.zeros(2, 3, 2, 48, device=DEV)[:, 1]):
        paged_attention(q, k, v, table, n, weights=apart)
        assert torch.equal(apart, plain)
    assert _status() == 0


def test_evict_outputs_must_not_reach_into_inputs():
    from dcr_b200.kernel.cuda.paged import paged_evict
    k, v, table, _, n = _small()
    both = torch.rand(2, 2, 2, 48, generator=_gen(4), device=DEV)
    ids = torch.arange(48, dtype=torch.int32, device=DEV).expand(2, 2, 48).contiguous()
    flat = both.view(-1)
    evict = lambda w, pos, **kw: paged_evict(k, v, table, n, w, pos, n, 20, **kw)  # noqa: E731
    for w, pos, kw in ((both[0], ids, dict(weights_out=flat[96:288].view(2, 2, 48))),
                       (both[:, 0], ids, dict(weights_out=both[:, 0, :, 8:])),
                       (both[0], ids, dict(weights_out=ids.view(torch.float32))),
                       (both[0], ids, dict(pos_out=both[0].view(torch.int32))),
                       (both[0], ids, dict(weights_out=both[1], pos_out=both[1].view(torch.int32)))):
        with pytest.raises(AssertionError, match="memory"):
            evict(w, pos, **kw)
    # between the rows of the inputs there is room
    want = paged_evict(k.clone(), v.clone(), table, n, both[:, 0].clone(), ids, n, 20)
    got = evict(both[:, 0], ids, weights_out=both[:, 1])
    assert torch.equal(got[1][:, :, :20], want[1]) and torch.equal(got[0], want[0])
    assert torch.equal(got[2], want[2]) and _status() == 0


def test_processed_logits_must_not_reach_into_the_logits():
    from dcr_b200.kernel.cuda.logits import process_logits
    flat = torch.randn(1000, generator=_gen(1), device=DEV)
    x = flat[:400].view(4, 100)
    for out in (flat[50:450].view(4, 100), flat[1:401].view(4, 100), flat[:800].view(4, 200)[:, :100]):
        with pytest.raises(AssertionError):
            process_logits(x, out=out)
    with pytest.raises(AssertionError):
        process_logits(flat[:100].expand(4, 100), out=x)
    want, token = process_logits(x.clone())
    wide = torch.zeros(4, 200, device=DEV)
    wide[:, 100:] = x
    got, t = process_logits(wide[:, 100:], out=wide[:, :100])
    assert torch.equal(got, want) and torch.equal(t, token)
    got, t = process_logits(x, out=x)
    assert torch.equal(got, want) and torch.equal(t, token) and _status() == 0


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_attention_and_append_in_place_or_apart(dt):
    from dcr_b200.kernel.cuda.paged import paged_append, paged_attention
    lengths = [3000, 0, 17, 900]
    k, v, table = ref.make_pool(lengths, 2, 16, 64, dt, DEV, _gen(5), garbage=0.0)
    packed = torch.randn(4, 24, 64, generator=_gen(6), device=DEV).to(dt)
    q = packed[:, :20].contiguous()
    x = q.clone()
    want = paged_attention(q, k, v, table, _i32(lengths))
    assert paged_attention(x, k, v, table, _i32(lengths), out=x) is x and torch.equal(x, want)
    cos = torch.rand(64, 64, generator=_gen(7), device=DEV).to(dt)
    append = lambda x, **kw: paged_append(x, packed[:, 20:22], packed[:, 22:], cos, cos, _i32([1, 2, 3, 4]),  # noqa: E731
                                          k, v, table, _i32([7, -1, 7, 7]), q_weight=cos[0], **kw)
    turned = append(q)
    into = packed.view(-1)[:4 * 20 * 64].view(4, 20, 64)  # contiguous, over the packed rows
    for call in (lambda: paged_attention(packed[:, :20], k, v, table, _i32(lengths), out=into),
                 lambda: append(packed[:, :20], out=into)):
        with pytest.raises(AssertionError, match="memory"):
            call()
    x = q.clone()
    assert append(x, out=x) is x and torch.equal(x, turned)
    assert _status() == 0


def _model(layers=2):
    from dcr_b200.models.llama.model import DCRLlamaDecoder, LlamaDecodeConfig
    cfg = LlamaDecodeConfig(vocab=512, hidden=256, intermediate=512, layers=layers, heads=4, kv_heads=2)
    return DCRLlamaDecoder(cfg, attention="dense", dtype=torch.float32, device=DEV, seed=0)


@pytest.mark.parametrize("slack", [1, 5])
def test_a_prompt_over_the_budget_keeps_what_its_last_token_attended_to(slack):
    from dcr_b200.models.llama.paged import PagedLlamaDecoder
    paged = PagedLlamaDecoder(_model(), max_positions=128)
    cache = paged.new_cache(3, 40, 128, page_size=8, budget=24, sinks=2, recent=4, slack=slack)
    g = torch.Generator().manual_seed(7)
    lengths = [60, 27, 10]
    plain, turned = cache.append, []
    cache.append = lambda *a, **kw: turned.append(plain(*a, **kw)) or turned[-1]
    paged.prefill([torch.randint(0, 512, (n,), generator=g).tolist() for n in lengths], cache)
    last = torch.tensor([59, 86, 96], device=DEV)
    W, tol = [], []
    for i in range(2):  # the definition, over what the pages hold; the third is not over the budget
        r = ref.attend(turned[i][last], cache.k[i], cache.v[i], cache.page_table, [60, 27, 0])
        W.append(r[2]), tol.append(r[5])
        assert ((cache.weights[i].double() - r[2]).abs() <= r[5]).all()
    paged.step(torch.tensor([1, 2, 3], device=DEV), cache)
    assert cache.host_lengths == [25, 25, 11]
    by_index = True
    for i in range(2):
        for b in range(2):
            n = lengths[b]
            for h in range(2):
                kept = set(cache.pos[i][b, h, :24].tolist())
                sure = set(range(2)) | set(range(n - 4, n))
                assert len(kept) == 24 and sure <= kept
                dropped = sorted(set(range(n)) - kept)
                least = min(float(W[i][b, h, p]) for p in kept - sure)
                most = max(float(W[i][b, h, p]) for p in dropped)
                assert least >= most - 2 * float(tol[i][b, h, :n].max())
                by_index &= kept == set(range(20)) | sure
    assert not by_index
    assert _status() == 0
