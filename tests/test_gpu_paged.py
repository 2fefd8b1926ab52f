"""The paged serving operators on the GPU against their definitions in 64 bits (paged_ref.py):
attention over pages, norms + rotation + append, eviction, at the sizes, layouts and masks where
they can go wrong, and their refusals."""
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
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _status():
    from dcr_b200 import _lib
    return _lib.read_device_status(clear=True)


def _lens(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _check_attention(lengths, H, H_kv, D, page, dt, *, seed=0, layout="hnd", window=0, unmap=(),
                     with_weights=True, scale=None, width=None, garbage=float("nan")):
    from dcr_b200.kernel.cuda.paged import paged_attention
    g = _gen(seed)
    k, v, table = ref.make_pool(lengths, H_kv, page, D, dt, DEV, g, layout=layout, width=width,
                                garbage=garbage)
    for b, i in unmap:
        table[b, i] = -1
    q = (2.0 * torch.randn(len(lengths), H, D, generator=g, device=DEV)).to(dt)
    w0 = torch.rand(len(lengths), H_kv, table.shape[1] * page, generator=g, device=DEV)
    w = w0.clone() if with_weights else None
    o, lse = paged_attention(q, k, v, table, _lens(lengths), window=window, weights=w, scale=scale,
                             return_lse=True)
    O, LSE, W, to, tl, tw = ref.attend(q, k, v, table, lengths, window, scale)
    assert ((o.double() - O).abs() <= to).all(), float(((o.double() - O).abs() / to).max())
    empty = LSE == -math.inf
    assert torch.equal(lse == -math.inf, empty) and (o[empty] == 0).all()
    assert ((lse.double() - LSE).abs() <= tl)[~empty].all()
    if with_weights:
        d = (w.double() - (w0.double() + W)).abs()
        assert (d <= tw + 2 * ref.EPS * (1 + w.double().abs())).all()
        assert torch.equal(w[W == 0], w0[W == 0])  # what no head attends to is not touched
    assert _status() == 0
    return o, lse, w


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,H_kv", [(1, 1), (6, 2), (4, 1), (16, 2), (24, 2), (16, 1), (40, 2)])
def test_attention_heads_and_types(dt, D, H, H_kv):
    _check_attention([0, 1, 2, 15, 16, 17, 63, 64, 65, 300], H, H_kv, D, 16, DT[dt])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 48, 64, 256])
def test_attention_page_sizes_and_layouts(dt, layout, page):
    _check_attention([257, 0, 100, 1, 511], 8, 2, 64, page, DT[dt], layout=layout, seed=page)


@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 5000])
def test_attention_window(dt, window):
    _check_attention([1, 16, 99, 100, 101, 700, 0], 8, 2, 64, 16, DT[dt], window=window, seed=window)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_attention_unmapped_pages(dt):
    # holes in the middle, at both ends, and a row whose every page is gone
    _check_attention([100, 64, 33, 48], 4, 2, 64, 16, DT[dt],
                     unmap=[(0, 0), (0, 3), (1, 3), (2, 0), (2, 1), (2, 2), (3, 1)])


@pytest.mark.parametrize("dt,D", [("bf16", 64), ("f16", 128), ("f32", 64)])
def test_attention_long_and_ragged(dt, D):
    _check_attention([20001, 3, 0, 7777, 12345], 8, 2, D, 64, DT[dt], with_weights=True, seed=4)


@pytest.mark.parametrize("B", [33, 300])
def test_attention_many_sequences(B):
    lengths = [(37 * b) % 90 for b in range(B)]
    _check_attention(lengths, 4, 2, 64, 16, torch.bfloat16, seed=B)


@pytest.mark.parametrize("garbage", [float("inf"), float("-inf"), float("nan")])
def test_attention_garbage_outside(garbage):
    _check_attention([5, 17, 40], 4, 4, 64, 32, torch.float16, garbage=garbage, window=11)


def test_attention_all_long_one_head():
    _check_attention([70000], 1, 1, 64, 64, torch.bfloat16, seed=9)


@pytest.mark.parametrize("dt", sorted(DT))
def test_attention_large_scores(dt):
    """Scores of several hundreds: the maximum grows along the row and the sum must not overflow."""
    from dcr_b200.kernel.cuda.paged import paged_attention
    n, D = 1000, 64
    k, v, table = ref.make_pool([n], 1, 16, D, DT[dt], DEV, _gen(3))
    q = torch.ones(1, 2, D, device=DEV).to(DT[dt])
    at = torch.arange(n, device=DEV)
    k[table[0, at // 16].long(), 0, at % 16] = (at / 16.0).floor()[:, None].expand(n, D).to(DT[dt])
    o, lse = paged_attention(q, k, v, table, _lens([n]), return_lse=True)
    O, LSE, _, to, tl, _ = ref.attend(q, k, v, table, [n])
    assert ((o.double() - O).abs() <= to).all() and ((lse.double() - LSE).abs() <= tl).all()


def test_attention_minus_infinity_scores_are_masked():
    from dcr_b200.kernel.cuda.paged import paged_attention
    k, v, table = ref.make_pool([20, 20], 1, 16, 64, torch.float32, DEV, _gen(5), garbage=0.0)
    q = torch.rand(2, 2, 64, device=DEV) + 0.5
    k[table[0, 0].long(), 0, :5] = -math.inf
    k[table[1].long()] = -math.inf
    o, lse = paged_attention(q, k, v, table, _lens([20, 20]), return_lse=True)
    k2 = k.clone()
    k2[table[0, 0].long(), 0, :5] = 0
    at = torch.arange(5, 20, device=DEV)
    z = (q[0].double() @ k2[table[0, at // 16].long(), 0, at % 16].double().T) / 8
    want = torch.softmax(z, -1) @ v[table[0, at // 16].long(), 0, at % 16].double()
    assert (o[0].double() - want).abs().max() < 1e-5
    assert (o[1] == 0).all() and (lse[1] == -math.inf).all()


def test_attention_strided_queries_and_out():
    from dcr_b200.kernel.cuda.paged import paged_attention, paged_workspace_bytes
    B, H, H_kv, D = 3, 8, 2, 64
    k, v, table = ref.make_pool([50, 20, 70], H_kv, 16, D, torch.bfloat16, DEV, _gen(6))
    qkv = torch.randn(B, H + 2 * H_kv, D, device=DEV).to(torch.bfloat16)
    want = paged_attention(qkv[:, :H].contiguous(), k, v, table, _lens([50, 20, 70]))
    out = torch.empty(B, H, D, device=DEV, dtype=torch.bfloat16)
    ws = torch.empty(paged_workspace_bytes(B, H, H_kv, D, table.shape[1] * 16), dtype=torch.uint8,
                     device=DEV)
    ws.fill_(255)
    got = paged_attention(qkv[:, :H], k, v, table, _lens([50, 20, 70]), out=out, workspace_buf=ws)
    assert got is out and torch.equal(got, want)
    wide = torch.full((B, table.shape[1] + 3), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    assert torch.equal(paged_attention(qkv[:, :H], k, v, wide[:, :table.shape[1]],
                                       _lens([50, 20, 70])), want)


def test_attention_is_deterministic_and_reuses_dirty_workspaces():
    from dcr_b200.kernel.cuda.paged import paged_attention, paged_workspace_bytes
    lengths = [5000, 1, 0, 999, 3000]
    k, v, table = ref.make_pool(lengths, 2, 16, 64, torch.bfloat16, DEV, _gen(7))
    q = torch.randn(5, 8, 64, device=DEV).to(torch.bfloat16)
    ws = torch.empty(paged_workspace_bytes(5, 8, 2, 64, table.shape[1] * 16, True), dtype=torch.uint8,
                     device=DEV)
    res = []
    for fill in (0, 255, 127):
        ws.fill_(fill)
        w = torch.zeros(5, 2, table.shape[1] * 16, device=DEV)
        res.append((*paged_attention(q, k, v, table, _lens(lengths), weights=w, return_lse=True,
                                     workspace_buf=ws), w))
    for r in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, res[0]))


def test_attention_on_another_stream_and_in_a_graph():
    from dcr_b200.kernel.cuda.paged import paged_attention
    cap = [600, 600]
    k, v, table = ref.make_pool(cap, 2, 16, 64, torch.bfloat16, DEV, _gen(8))
    q = torch.randn(2, 8, 64, device=DEV).to(torch.bfloat16)
    n = _lens([100, 300])
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        paged_attention(q, k, v, table, n, out=out)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            paged_attention(q, k, v, table, n, out=out)
    for lengths in ([100, 300], [600, 0], [1, 599]):
        n.copy_(_lens(lengths))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        O, _, _, to, _, _ = ref.attend(q, k, v, table, lengths)
        assert ((out.double() - O).abs() <= to).all()


def test_attention_past_32_bit_offsets():
    """A pool of more than 2^31 elements: the last pages are addressed in 64 bits."""
    from dcr_b200.kernel.cuda.paged import paged_append, paged_attention
    page, H_kv, D = 64, 8, 64
    pages = (1 << 31) // (page * H_kv * D) + 70
    k = torch.empty(pages, H_kv, page, D, dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    table = torch.arange(pages - 4, pages, dtype=torch.int32, device=DEV).view(1, 4)
    k[-4:] = torch.randn(4, H_kv, page, D, generator=_gen(1), device=DEV).to(k.dtype)
    v[-4:] = torch.randn(4, H_kv, page, D, generator=_gen(2), device=DEV).to(k.dtype)
    q = torch.randn(1, 32, D, generator=_gen(3), device=DEV).to(k.dtype)
    O, _, _, to, _, _ = ref.attend(q, k, v, table, [250])
    assert ((paged_attention(q, k, v, table, _lens([250])).double() - O).abs() <= to).all()
    x = torch.randn(1, H_kv, D, device=DEV).to(k.dtype)
    one, zero = torch.ones(1, D, device=DEV), torch.zeros(1, D, device=DEV)
    paged_append(q, x, x, one, zero, _lens([0]), k, v, table, _lens([250]))
    assert torch.equal(k[-1, :, 250 % 64], x[0]) and torch.equal(v[-1, :, 250 % 64], x[0])
    del k, v
    torch.cuda.empty_cache()


def test_entries_out_of_range_are_skipped_and_reported():
    from dcr_b200 import _lib
    from dcr_b200.kernel.cuda.paged import paged_attention
    k, v, table = ref.make_pool([40, 40], 2, 16, 64, torch.bfloat16, DEV, _gen(2))
    q = torch.randn(2, 4, 64, device=DEV).to(torch.bfloat16)
    bad = table.clone()
    bad[0, 1] = k.shape[0]
    O, _, _, to, _, _ = ref.attend(q, k, v, torch.where(bad >= k.shape[0], -1, bad), [40, 40])
    assert _status() == 0
    o = paged_attention(q, k, v, bad, _lens([40, 40]))
    assert ((o.double() - O).abs() <= to).all() and _status() == _lib.DCR_ERR_DEVICE_INDEX
    # a length past the table's slots is held to them, a negative one is 0
    full, _, _, to, _, _ = ref.attend(q, k, v, table, [48, 0])
    k[table[0, 2].long(), :, 8:] = 0
    v[table[0, 2].long(), :, 8:] = 0
    full, _, _, to, _, _ = ref.attend(q, k, v, table, [48, 0])
    o = paged_attention(q, k, v, table, _lens([1 << 30, -5]))
    assert ((o.double() - full).abs() <= to).all() and _status() == _lib.DCR_ERR_DEVICE_INDEX


# ------------------------------------------------------------------------------- norms and append
def _tables(n, D, dt):
    a = torch.arange(n, device=DEV).double()[:, None] * 10000.0 ** (
        -torch.arange(0, D, 2, device=DEV).double() / D)
    a = torch.cat((a, a), 1)
    return a.cos().to(dt), a.sin().to(dt)


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,H,H_kv", [(1, 1, 1), (1, 32, 8), (5, 6, 2), (130, 12, 4)])
@pytest.mark.parametrize("norm,f32_tables,layout", [(True, False, "hnd"), (False, True, "nhd"),
                                                    (True, True, "hnd")])
def test_append(dt, D, T, H, H_kv, norm, f32_tables, layout):
    from dcr_b200.kernel.cuda.paged import paged_append
    t = DT[dt]
    g = _gen(T + D)
    page, parts = 24, [T // 2, 0, T - T // 2]
    k, v, table = ref.make_pool([n + 30 for n in parts], H_kv, page, D, t, DEV, g, layout=layout)
    seq = [b for b, n in enumerate(parts) for _ in range(n)]
    slots = [i + 30 for n in parts for i in range(n)]
    if T > 4:
        slots[3] = -1  # a token that is not kept
    positions = [(13 * i) % 200 for i in range(T)]
    qkv = torch.randn(T, H + 2 * H_kv, D, generator=g, device=DEV).to(t)
    if T > 2:
        qkv[2] = 0  # a row of zeros: its norm is eps
    qw = torch.randn(D, generator=g, device=DEV).to(t) if norm else None
    kw = torch.randn(D, generator=g, device=DEV).to(t) if norm else None
    cos, sin = _tables(200, D, torch.float32 if f32_tables else t)
    cap = table.shape[1] * page
    w = torch.full((3, H_kv, cap), 5.0, device=DEV)
    pos = torch.full((3, H_kv, cap), -7, dtype=torch.int32, device=DEV)
    k0, v0 = k.clone(), v.clone()
    out = paged_append(qkv[:, :H], qkv[:, H:H + H_kv], qkv[:, H + H_kv:], cos, sin, _lens(positions),
                       k, v, table, _lens(slots), seq=_lens(seq), q_weight=qw, k_weight=kw, eps=1e-6,
                       weights=w, pos=pos)
    p = torch.tensor(positions, device=DEV)
    Q, tq = ref.norm_rotate(qkv[:, :H], qw, cos[p], sin[p], 1e-6, t)
    K, tk = ref.norm_rotate(qkv[:, H:H + H_kv], kw, cos[p], sin[p], 1e-6, t)
    assert ((out.double() - Q).abs() <= tq).all()
    keep = [i for i in range(T) if slots[i] >= 0]
    sq, sl = torch.tensor(seq, device=DEV)[keep], torch.tensor(slots, device=DEV)[keep]
    pg = table[sq, sl // page].long()
    assert ((k[pg, :, sl % page].double() - K[keep]).abs() <= tk[keep]).all()
    assert torch.equal(v[pg, :, sl % page], qkv[keep][:, H + H_kv:])
    k[pg, :, sl % page] = k0[pg, :, sl % page]
    v[pg, :, sl % page] = v0[pg, :, sl % page]
    assert torch.equal(k.nan_to_num(9), k0.nan_to_num(9)) and torch.equal(v.nan_to_num(9), v0.nan_to_num(9))
    hit = torch.zeros(3, cap, dtype=torch.bool, device=DEV)
    hit[sq, sl] = True
    assert (w.transpose(1, 2)[hit] == 0).all() and (w.transpose(1, 2)[~hit] == 5).all()
    assert (pos.transpose(1, 2)[~hit] == -7).all()
    assert torch.equal(pos[sq, 0, sl].long(), p[keep]) and torch.equal(pos[sq, -1, sl].long(), p[keep])
    assert _status() == 0


def test_append_without_seq_and_empty():
    from dcr_b200.kernel.cuda.paged import paged_append
    k, v, table = ref.make_pool([40, 40], 2, 16, 64, torch.bfloat16, DEV, _gen(2))
    x = torch.randn(2, 8, 64, device=DEV).to(torch.bfloat16)
    cos, sin = _tables(64, 64, torch.bfloat16)
    out = paged_append(x[:, :4], x[:, 4:6], x[:, 6:], cos, sin, _lens([3, 9]), k, v, table, _lens([39, 7]))
    assert torch.equal(v[table[1, 0].long(), :, 7], x[1, 6:]) and out.shape == (2, 4, 64)
    none = paged_append(x[:0, :4], x[:0, 4:6], x[:0, 6:], cos, sin, _lens([]), k, v, table, _lens([]))
    assert none.shape == (0, 4, 64)


def test_append_reports_what_it_cannot_place():
    from dcr_b200 import _lib
    from dcr_b200.kernel.cuda.paged import paged_append
    k, v, table = ref.make_pool([20, 20], 1, 16, 64, torch.float32, DEV, _gen(2), width=3)
    x = torch.randn(2, 3, 64, device=DEV)
    cos, sin = _tables(8, 64, torch.float32)
    k0 = k.clone().nan_to_num(9)
    args = lambda p, s, **kw: paged_append(x[:, :1], x[:, 1:2], x[:, 2:], cos, sin, _lens(p), k, v,  # noqa: E731
                                           table, _lens(s), **kw)
    assert _status() == 0
    out = args([8, -1], [0, 0])                       # positions past the tables
    assert (out == 0).all() and _status() == _lib.DCR_ERR_DEVICE_INDEX
    args([1, 1], [48, 40])                            # past the slots; in an unmapped page
    assert _status() == _lib.DCR_ERR_DEVICE_INDEX
    args([1, 1], [0, 0], seq=_lens([2, -1]))          # no such sequences
    assert _status() == _lib.DCR_ERR_DEVICE_INDEX
    assert torch.equal(k.nan_to_num(9), k0)


# ----------------------------------------------------------------------------------------- eviction
def _check_evict(lengths, H_kv, budget, page, dt, *, D=64, sinks=0, recent=0, layout="hnd", seed=0,
                 make=None, width=None):
    from dcr_b200.kernel.cuda.paged import paged_evict
    g = _gen(seed)
    B = len(lengths)
    k, v, table = ref.make_pool(lengths, H_kv, page, D, dt, DEV, g, layout=layout, width=width)
    cap = table.shape[1] * page
    w = torch.rand(B, H_kv, cap, generator=g, device=DEV)
    pos = torch.rand(B, H_kv, cap, generator=g, device=DEV).argsort(-1).to(torch.int32)
    if make is not None:
        make(w, pos)
    seen = _lens([cap] * B)
    n = _lens(lengths)
    k0, v0, w0, p0 = k.clone(), v.clone(), w.clone(), pos.clone()
    src, wo, po, no = paged_evict(k, v, table, n, w, pos, seen, budget, sinks=sinks, recent=recent)
    assert torch.equal(w.nan_to_num(9), w0.nan_to_num(9)) and torch.equal(pos, p0)
    assert no.tolist() == [min(x, budget) for x in lengths]
    want = torch.tensor([[ref.evict(w0[b, h, :lengths[b]].tolist(), p0[b, h, :lengths[b]].tolist(),
                                    lengths[b], cap, budget, sinks, recent) for h in range(H_kv)]
                         for b in range(B)], dtype=torch.int32, device=DEV)
    assert torch.equal(src, want)
    held = want >= 0
    at = want.long().clamp(min=0)
    assert torch.equal(wo.nan_to_num(9), torch.where(held, w0.gather(2, at), 0.0).nan_to_num(9))
    assert torch.equal(po, torch.where(held, p0.gather(2, at), -1))
    b, h, i = torch.nonzero(held, as_tuple=True)
    s = at[b, h, i]
    fp, tp = table[b, s // page].long(), table[b, i // page].long()
    for new, old in ((k, k0), (v, v0)):
        expect = old.clone()
        expect[tp, h, i % page] = old[fp, h, s % page]
        assert torch.equal(new.nan_to_num(9), expect.nan_to_num(9))
    assert _status() == 0


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("layout,page", [("hnd", 16), ("nhd", 5)])
def test_evict_types_and_layouts(dt, D, layout, page):
    _check_evict([100, 0, 1, 33, 31, 32], 2, 32, page, DT[dt], D=D, layout=layout, sinks=2, recent=9)


@pytest.mark.parametrize("n,budget", [(2, 1), (1000, 1), (1000, 999), (1025, 1024), (5000, 2500),
                                      (20000, 3000), (40000, 39999), (9000, 8997), (1004, 1000), (1005, 1000), (36000, 35998), (1000, 1000)])
def test_evict_sizes(n, budget):
    _check_evict([n, max(1, n // 2)], 2, budget, 64, torch.bfloat16, sinks=4, recent=budget // 4, seed=n)


def test_evict_rows_that_registers_cannot_hold():
    _check_evict([300001], 1, 1000, 64, torch.bfloat16, sinks=1, recent=100)


@pytest.mark.parametrize("few", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("n", [40, 3000, 20000])
def test_evict_few(few, n):
    """The evicted ones at the front, at the end (no move at all) and among ties."""
    for make in (None, _ties, _zeros, _wild, lambda w, pos: w[..., -n:].copy_(-torch.arange(n, device=DEV)),
                 lambda w, pos: w.copy_(torch.arange(w.shape[-1], device=DEV))):
        _check_evict([n, n - 1], 2, n - few, 16, torch.bfloat16, make=make, recent=3, sinks=1)


def _ties(w, pos):
    w.mul_(4).floor_()


def _zeros(w, pos):
    w.zero_()
    w[..., 1::2] = -0.0


def _wild(w, pos):
    w[..., ::7] = float("nan")
    w[..., 1::7] = float("inf")
    w[..., 2::7] = float("-inf")
    w[..., 3::7] *= -1
    w[..., 4::7] *= 1e-40


@pytest.mark.parametrize("make", [_ties, _zeros, _wild])
@pytest.mark.parametrize("n", [300, 3001])
def test_evict_ties_and_odd_values(make, n):
    _check_evict([n, n - 7], 3, n // 3, 16, torch.float16, make=make, recent=5)


@pytest.mark.parametrize("sinks,recent", [(0, 2000), (2000, 0), (90, 90), (0, 1)])
def test_evict_protected(sinks, recent):
    """More protected slots than the budget: the lowest slots of them stay."""
    _check_evict([700, 100, 50], 2, 60, 16, torch.bfloat16, sinks=sinks, recent=recent)


def test_evict_one_step_at_a_time():
    """Steady state: a slot over the budget each step, the table of the step before goes in."""
    from dcr_b200.kernel.cuda.paged import paged_evict
    budget, page = 20, 8
    k, v, table = ref.make_pool([budget + 1], 1, page, 64, torch.float32, DEV, _gen(1))
    g = _gen(2)
    cap = table.shape[1] * page
    w = torch.rand(1, 1, cap, generator=g, device=DEV)
    pos = torch.arange(cap, dtype=torch.int32, device=DEV).view(1, 1, cap).clone()
    spare_w, spare_p = torch.zeros_like(w), torch.zeros_like(pos)
    rows = {i: k[table[0, i // page].long(), 0, i % page].clone() for i in range(budget + 1)}
    n = _lens([budget + 1])
    for step in range(40):
        before = {int(p): float(x) for p, x in zip(pos[0, 0, :budget + 1].tolist(), w[0, 0, :budget + 1].tolist())}
        seen = budget + 1 + step
        paged_evict(k, v, table, n, w, pos, _lens([seen]), budget, sinks=1, recent=4,
                    weights_out=spare_w, pos_out=spare_p)
        w, spare_w, pos, spare_p = spare_w, w, spare_p, pos
        left = set(pos[0, 0, :budget].tolist())
        free = {p: x for p, x in before.items() if 1 <= p < seen - 4}
        assert set(before) - left == {min(free, key=free.get)}
        for i in range(budget):
            assert torch.equal(k[table[0, i // page].long(), 0, i % page], rows[int(pos[0, 0, i])])
        new = torch.randn(64, generator=g, device=DEV)  # the next step's slot
        k[table[0, budget // page].long(), 0, budget % page] = new
        rows[seen] = new
        w[0, 0, budget], pos[0, 0, budget] = torch.rand(1, generator=g, device=DEV)[0], seen


# ----------------------------------------------------------------------------------------- refusals
def test_refusals():
    from dcr_b200.kernel.cuda.paged import paged_append, paged_attention, paged_evict
    k, v, table = ref.make_pool([40, 40], 2, 16, 64, torch.bfloat16, DEV, _gen(2))
    q = torch.randn(2, 4, 64, device=DEV).to(torch.bfloat16)
    n = _lens([40, 40])
    ok = dict(q=q, k_pages=k, v_pages=v, page_table=table, lengths=n)
    for change in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[:, :, :32]), dict(q=q[:1]),
                   dict(v_pages=v[:, :1]), dict(v_pages=v.half()), dict(k_pages=k[..., :32], v_pages=v[..., :32]),
                   dict(page_table=table.long()), dict(page_table=table[:1]), dict(lengths=n.long()),
                   dict(lengths=_lens([1])), dict(window=-1), dict(weights=torch.zeros(2, 2, 40, device=DEV)),
                   dict(weights=torch.zeros(2, 2, 48, device=DEV).double()),
                   dict(out=torch.empty(2, 4, 64, device=DEV)), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)),
                   dict(workspace_buf=torch.empty(0, dtype=torch.uint8, device=DEV))):
        with pytest.raises(AssertionError):
            paged_attention(**{**ok, **change})
    for change in (dict(q=q.cpu()), dict(k_pages=k.cpu()), dict(lengths=n.cpu())):
        with pytest.raises(RuntimeError):
            paged_attention(**{**ok, **change})
    base = torch.empty(2 * 4 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(2, 4, 64)
    with pytest.raises(RuntimeError, match="dcr_status 5"):  # rows off a 16-byte boundary
        paged_attention(**{**ok, "q": base})
    cos, sin = _tables(8, 64, torch.bfloat16)
    ap = dict(q=q, k=q[:, :2], v=q[:, 2:], cos=cos, sin=sin, positions=n, k_pages=k, v_pages=v,
              page_table=table, slots=n)
    for change in (dict(k=q), dict(cos=cos.half()), dict(sin=sin[:4]), dict(positions=n.long()),
                   dict(slots=n[:1]), dict(q_weight=torch.ones(64, device=DEV)), dict(seq=n[:1]),
                   dict(k_weight=torch.ones(32, device=DEV).to(torch.bfloat16)),
                   dict(pos=torch.zeros(2, 2, 48, device=DEV))):
        with pytest.raises(AssertionError):
            paged_append(**{**ap, **change})
    w = torch.zeros(2, 2, 48, device=DEV)
    p = torch.zeros(2, 2, 48, dtype=torch.int32, device=DEV)
    ev = dict(k_pages=k, v_pages=v, page_table=table, lengths=n, weights=w, pos=p, seen=n, budget=20)
    for change in (dict(budget=0), dict(budget=49), dict(sinks=-1), dict(recent=-1), dict(weights=w[:, :1]),
                   dict(pos=p.long()), dict(seen=n[:1]), dict(weights_out=w), dict(pos_out=p)):
        with pytest.raises(AssertionError):
            paged_evict(**{**ev, **change})
