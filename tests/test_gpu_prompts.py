"""Prompts, shared prefixes and rotations on the GPU against their definitions in 64 bits (rows_ref.py),
at the sizes, layouts and masks where they can go wrong, and their refusals."""
from __future__ import annotations

import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_ref  # noqa: E402
import rows_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _status():
    from dcr_b200 import _lib
    return _lib.read_device_status(clear=True)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _starts(news):
    out = [0]
    for n in news:
        out.append(out[-1] + n)
    return out


# -------------------------------------------------------------------------------------- prefill
def _compare(o, lse, want, nans=None):
    O, LSE, to, tl = want
    d = (o.double() - O).abs()
    if nans is not None:
        assert torch.equal(torch.isnan(o).all(-1), nans) and torch.equal(torch.isnan(o).any(-1), nans)
        d = torch.where(nans[..., None], 0.0, d)
    assert (d <= to).all(), float((d / to).max())
    empty = LSE == -math.inf
    assert torch.equal(lse == -math.inf, empty) and (o[empty] == 0).all()
    assert ((lse.double() - LSE).abs() <= tl)[~empty].all()


def _check_prefill(news, lengths, H, H_kv, D, page, dt, *, seed=0, layout="hnd", window=0, causal=True,
                   unmap=(), scale=None, width=None, garbage=float("nan"), q_scale=2.0):
    from dcr_b200.kernel.cuda import paged_prefill
    g = _gen(seed)
    k, v, table = paged_ref.make_pool(lengths, H_kv, page, D, dt, DEV, g, layout=layout, width=width,
                                      garbage=garbage)
    for b, i in unmap:
        table[b, i] = -1
    starts = _starts(news)
    q = (q_scale * torch.randn(starts[-1], H, D, generator=g, device=DEV)).to(dt)
    o, lse = paged_prefill(q, k, v, table, _i32(lengths), _i32(starts), window=window, causal=causal,
                           scale=scale, return_lse=True)
    lo, hi, seq = ref.prefill_limits(starts, lengths, window, causal)
    want = ref.attend(q, k, v, table[seq], lo, hi, scale=scale,
                      weight_unit=0.0 if dt == torch.float32 else paged_ref.UNIT[dt])
    _compare(o, lse, want)
    assert _status() == 0
    return q, k, v, table, o, lse


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,H_kv", [(1, 1), (6, 2), (4, 1), (16, 2), (10, 2), (16, 1), (24, 1), (3, 3)])
def test_prefill_heads_and_types(dt, D, H, H_kv):
    _check_prefill([1, 0, 5, 64, 33, 130], [1, 9, 5, 64, 300, 131], H, H_kv, D, 16, DT[dt])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 48, 64, 100, 256])
def test_prefill_page_sizes_and_layouts(dt, layout, page):
    _check_prefill([200, 0, 7, 129], [257, 100, 511, 129], 8, 2, 64, page, DT[dt], layout=layout, seed=page)


@pytest.mark.parametrize("dt,D", [("f16", 64), ("bf16", 128), ("f32", 64)])
@pytest.mark.parametrize("window", [1, 2, 16, 127, 128, 129, 300, 5000])
def test_prefill_window(dt, D, window):
    _check_prefill([100, 400, 3, 1], [100, 700, 513, 129], 8, 2, D, 16, DT[dt], window=window, seed=window)


@pytest.mark.parametrize("dt", sorted(DT))
def test_prefill_not_causal(dt):
    _check_prefill([40, 1, 0, 129], [200, 1, 50, 129], 8, 2, 64, 16, DT[dt], causal=False)


@pytest.mark.parametrize("dt", sorted(DT))
def test_prefill_unmapped_pages(dt):
    # holes in the middle, at both ends, and a sequence whose every page is gone: its rows see nothing
    _check_prefill([100, 64, 33, 48], [300, 64, 33, 48], 4, 2, 64, 16, DT[dt],
                   unmap=[(0, 0), (0, 3), (0, 18), (1, 3), (2, 0), (2, 1), (2, 2), (3, 1)])


@pytest.mark.parametrize("dt,D", [("bf16", 64), ("f16", 128), ("f32", 64), ("bf16", 128), ("f16", 64)])
def test_prefill_long_history(dt, D):
    _check_prefill([5, 1, 300, 0], [20001, 7777, 12345, 3], 8, 2, D, 64, DT[dt], seed=4)


@pytest.mark.parametrize("dt,D", [("bf16", 64), ("f16", 128), ("f32", 128)])
def test_prefill_long_prompt(dt, D):
    _check_prefill([1999], [1999], 4, 1, D, 64, DT[dt], seed=5)


@pytest.mark.parametrize("B", [33, 300])
def test_prefill_many_sequences(B):
    news = [(5 * b) % 9 for b in range(B)]
    _check_prefill(news, [n + (37 * b) % 90 for b, n in enumerate(news)], 4, 2, 64, 16, torch.bfloat16, seed=B)


@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("garbage", [float("inf"), float("-inf"), float("nan")])
def test_prefill_garbage_outside(dt, garbage):
    _check_prefill([5, 17, 40], [5, 170, 41], 4, 4, 64, 32, DT[dt], garbage=garbage, window=11)


def test_prefill_scale_and_wide_table():
    _check_prefill([70], [333], 4, 2, 64, 16, torch.bfloat16, scale=0.03, width=500)


def _filled(n, H_kv, D, page, dt, seed):
    """One sequence's pool without spare slots, so that every slot can be named by its number."""
    k, v, table = paged_ref.make_pool([n], H_kv, page, D, dt, DEV, _gen(seed))
    at = torch.arange(n, device=DEV)
    return k, v, table, table[0, at // page].long(), at % page


@pytest.mark.parametrize("dt", sorted(DT))
def test_prefill_large_scores(dt):
    """Scores of several hundreds that grow along the row: the base must follow, sums not overflow."""
    from dcr_b200.kernel.cuda import paged_prefill
    n, D = 1000, 64
    k, v, table, pg, at = _filled(n, 1, D, 16, DT[dt], 3)
    k[pg, 0, at] = (torch.arange(n, device=DEV) / 16.0).floor()[:, None].expand(n, D).to(DT[dt])
    q = torch.ones(300, 2, D, device=DEV).to(DT[dt])
    o, lse = paged_prefill(q, k, v, table, _i32([n]), _i32([0, 300]), return_lse=True)
    lo, hi, seq = ref.prefill_limits([0, 300], [n], 0, True)
    unit = 0.0 if dt == "f32" else paged_ref.UNIT[DT[dt]]
    _compare(o, lse, ref.attend(q, k, v, table[seq], lo, hi, weight_unit=unit))


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", [float("inf"), float("-inf"), float("nan")])
def test_prefill_values_that_some_rows_do_not_see(dt, D, what):
    """A value that is not finite spoils the rows that see its slot and no others."""
    from dcr_b200.kernel.cuda import paged_prefill
    n, H, H_kv = 400, 4, 2
    k, v, table, pg, at = _filled(n, H_kv, D, 16, DT[dt], 7)
    q = torch.randn(n, H, D, generator=_gen(8), device=DEV).to(DT[dt])
    bad = [(130, 1, 3), (131, 1, 60), (299, 0, D - 1)]  # (slot, KV head, element)
    for s, h, d in bad:
        v[pg[s], h, at[s], d] = what
    window = 90
    o, lse = paged_prefill(q, k, v, table, _i32([n]), _i32([0, n]), window=window, return_lse=True)
    lo, hi, seq = ref.prefill_limits([0, n], [n], window, True)
    unit = 0.0 if dt == "f32" else paged_ref.UNIT[DT[dt]]
    O, LSE, to, tl = ref.attend(q, k, v, table[seq], lo, hi, weight_unit=unit)
    spoilt = torch.zeros(n, H, dtype=torch.bool, device=DEV)
    for s, h, _ in bad:
        spoilt[s:s + window, h * 2:h * 2 + 2] = True
    clean = ~spoilt
    assert ((o.double() - O).abs() <= to)[clean].all()
    assert not torch.isfinite(o[spoilt]).all(-1).any()
    assert ((lse.double() - LSE).abs() <= tl).all()


@pytest.mark.parametrize("dt", sorted(DT))
def test_prefill_keys_that_some_rows_do_not_see(dt):
    from dcr_b200.kernel.cuda import paged_prefill
    n = 200
    k, v, table, pg, at = _filled(n, 1, 64, 16, DT[dt], 9)
    q = torch.randn(n, 2, 64, generator=_gen(10), device=DEV).to(DT[dt])
    k[pg[150], 0, at[150]] = float("nan")
    o = paged_prefill(q, k, v, table, _i32([n]), _i32([0, n]))
    assert torch.isfinite(o[:150]).all() and torch.isnan(o[150:]).all()


@pytest.mark.parametrize("dt", sorted(DT))
def test_prefill_rows_of_nobody_and_tokens_before_the_cache(dt):
    from dcr_b200.kernel.cuda import paged_prefill
    g = _gen(11)
    k, v, table = paged_ref.make_pool([40, 20], 2, 16, 64, DT[dt], DEV, g)
    q = torch.randn(100, 4, 64, generator=g, device=DEV).to(DT[dt])
    out = torch.full((100, 4, 64), 7.0, device=DEV).to(DT[dt])
    got = paged_prefill(q, k, v, table, _i32([40, 20]), _i32([3, 33, 60]), out=out)
    assert got is out or got.data_ptr() == out.data_ptr()
    assert (out[:3] == 7).all() and (out[60:] == 7).all()
    assert (out[33:40] == 0).all()  # 27 tokens of a sequence of 20 slots: the first 7 see nothing
    lo, hi, seq = ref.prefill_limits([3, 33, 60], [40, 20], 0, True)
    unit = 0.0 if dt == "f32" else paged_ref.UNIT[DT[dt]]
    O, _, to, _ = ref.attend(q[3:60], k, v, table[seq], lo, [max(h, 0) for h in hi], weight_unit=unit)
    assert ((out[3:60].double() - O).abs() <= to).all() and _status() == 0


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_prefill_strided_queries_in_place_and_streams(dt):
    from dcr_b200.kernel.cuda import paged_prefill
    q, k, v, table, o, lse = _check_prefill([50, 20], [90, 200], 8, 2, 64, 16, DT[dt], seed=12)
    args = (k, v, table, _i32([90, 200]), _i32([0, 50, 70]))
    packed = torch.zeros(70, 12, 64, dtype=DT[dt], device=DEV)
    packed[:, 2:10] = q
    assert torch.equal(paged_prefill(packed[:, 2:10], *args), o)
    same = q.clone()
    assert torch.equal(paged_prefill(same, *args, out=same), o)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = paged_prefill(q, *args)
    side.synchronize()
    assert torch.equal(other, o)


def test_prefill_one_token_is_decode():
    from dcr_b200.kernel.cuda import paged_attention, paged_prefill
    lengths = [1, 17, 300, 0]
    k, v, table = paged_ref.make_pool(lengths, 2, 16, 64, torch.float32, DEV, _gen(13))
    q = torch.randn(4, 8, 64, generator=_gen(14), device=DEV)
    a = paged_attention(q, k, v, table, _i32(lengths))
    b = paged_prefill(q, k, v, table, _i32(lengths), _i32([0, 1, 2, 3, 4]))
    # sums of 300 terms in another order
    assert (a - b).abs().max() <= 2 * 300 * paged_ref.EPS * v[torch.isfinite(v)].abs().max() and _status() == 0


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_prefill_captured_and_replayed(dt):
    """Lengths, starts, table and queries may change between replays."""
    from dcr_b200.kernel.cuda import paged_prefill
    g = _gen(15)
    k, v, table = paged_ref.make_pool([500, 400], 2, 16, 64, DT[dt], DEV, g)
    q = torch.randn(64, 8, 64, generator=g, device=DEV).to(DT[dt])
    lengths, starts = _i32([100, 30]), _i32([0, 40, 64])
    paged_prefill(q, k, v, table, lengths, starts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = paged_prefill(q, k, v, table, lengths, starts)
    for n, s in [([100, 30], [0, 40, 64]), ([500, 399], [0, 1, 64]), ([64, 0], [0, 64, 64])]:
        lengths.copy_(_i32(n)), starts.copy_(_i32(s))
        q.copy_(torch.randn(64, 8, 64, generator=g, device=DEV).to(DT[dt]))
        graph.replay()
        want = paged_prefill(q, k, v, table, lengths, starts)
        assert torch.equal(o, want)


def test_prefill_bad_device_values():
    """Lengths past the table, pages past the pool and starts out of order are skipped and reported."""
    from dcr_b200.kernel.cuda import paged_prefill
    k, v, table = paged_ref.make_pool([40, 20], 1, 16, 64, torch.bfloat16, DEV, _gen(16))
    q = torch.randn(30, 2, 64, device=DEV).to(torch.bfloat16)
    run = lambda n, s, t=table: paged_prefill(q, k, v, t, _i32(n), _i32(s))  # noqa: E731
    run([1000, 20], [0, 20, 30])
    assert _status() != 0
    broken = table.clone()
    broken[0, 1] = 1 << 20
    run([40, 20], [0, 20, 30], broken)
    assert _status() != 0
    for starts in ([0, 25, 10], [-5, 10, 30], [0, 10, 31]):
        run([40, 20], starts)
        assert _status() != 0
    o = run([40, -3], [0, 20, 30])  # a negative length is an empty sequence
    assert (o[20:] == 0).all() and _status() == 0


def test_prefill_far_pages():
    """Element offsets past 32 bits."""
    from dcr_b200.kernel.cuda import paged_prefill
    pages, H_kv, page, D = 40000, 8, 64, 128  # 2.6e9 elements
    pool = torch.empty(pages, H_kv, page, D, dtype=torch.bfloat16, device=DEV)
    near = torch.randn(3, H_kv, page, D, generator=_gen(17), device=DEV).to(torch.bfloat16)
    pool[pages - 3:] = near
    q = torch.randn(70, 16, D, generator=_gen(18), device=DEV).to(torch.bfloat16)
    far, close = _i32([[pages - 1, pages - 3, pages - 2]]), _i32([[2, 0, 1]])
    a = paged_prefill(q, pool, pool, far, _i32([170]), _i32([0, 70]))
    b = paged_prefill(q, near, near, close, _i32([170]), _i32([0, 70]))
    assert torch.equal(a, b)


def test_prefill_refusals():
    from dcr_b200.kernel.cuda import paged_prefill
    k, v, table = paged_ref.make_pool([40, 20], 2, 16, 64, torch.bfloat16, DEV, _gen(19))
    q = torch.randn(30, 4, 64, device=DEV).to(torch.bfloat16)
    n, s = _i32([40, 20]), _i32([0, 20, 30])
    good = dict(q=q, k_pages=k, v_pages=v, page_table=table, lengths=n, starts=s)
    paged_prefill(**good)
    for bad in (dict(q=q[:, :3]), dict(q=q.float()), dict(q=q[..., :32]), dict(lengths=n[:1]),
                dict(starts=s[:2]), dict(starts=s.long()), dict(window=-1), dict(window=4, causal=False),
                dict(page_table=table.long()), dict(v_pages=v[:1]), dict(out=torch.empty_like(q)[:20]),
                dict(out=torch.empty(30, 4, 64, device=DEV)),
                dict(workspace_buf=torch.empty(3, dtype=torch.uint8, device=DEV))):
        with pytest.raises(AssertionError):
            paged_prefill(**dict(good, **bad))
    both = torch.empty(31, 4, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(AssertionError):
        paged_prefill(**dict(good, q=both[1:], out=both[:30]))
    with pytest.raises(RuntimeError):
        paged_prefill(**dict(good, starts=s.cpu()))
    assert paged_prefill(**dict(good, q=q[:0], starts=_i32([0, 0, 0]))).shape == (0, 4, 64)


# -------------------------------------------------------------------------------------- shared
def _make_shared(members, prefixes, owns, H_kv, page, D, dt, seed, layout="hnd"):
    """Groups whose sequences' first pages are the first sequence's: (k, v, table, lengths, prefix,
    groups)."""
    held, lengths, prefix, groups, first = [], [], [], [0], 0
    for m, pre in zip(members, prefixes):
        for i in range(m):
            own = owns[first + i]
            whole = pre // page * page  # pages that can be shared
            held.append(pre + own if i == 0 else pre + own - whole)
            lengths.append(pre + own)
            prefix.append(whole)
        first += m
        groups.append(first)
    width = max(-(-n // page) for n in lengths)
    k, v, own_table = paged_ref.make_pool(held, H_kv, page, D, dt, DEV, _gen(seed), layout=layout, width=width)
    table = own_table.clone()
    for g, a in enumerate(groups[:-1]):
        c = prefix[a] // page
        for b in range(a + 1, groups[g + 1]):
            table[b] = torch.cat((own_table[a, :c], own_table[b, :width - c]))
    return k, v, table, lengths, prefix, groups


def _check_shared(members, prefixes, owns, H, H_kv, D, page, dt, *, seed=0, window=0, layout="hnd", scale=None):
    from dcr_b200.kernel.cuda import paged_shared_attention
    k, v, table, lengths, prefix, groups = _make_shared(members, prefixes, owns, H_kv, page, D, dt, seed, layout)
    q = (2.0 * torch.randn(len(lengths), H, D, generator=_gen(seed + 1), device=DEV)).to(dt)
    o, lse = paged_shared_attention(q, k, v, table, _i32(lengths), _i32(groups), _i32(prefix), window=window,
                                    scale=scale, return_lse=True)
    lo = [max(0, n - window) if window else 0 for n in lengths]
    want = ref.attend(q, k, v, table, lo, lengths, scale=scale,
                      weight_unit=0.0 if dt == torch.float32 else 2.0 ** -16)
    _compare(o, lse, want)
    assert _status() == 0
    return q, k, v, table, lengths, prefix, groups, o


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,H_kv", [(1, 1), (6, 2), (16, 2), (5, 1), (32, 2)])
def test_shared_heads_and_types(dt, D, H, H_kv):
    _check_shared([3, 1, 20], [100, 40, 333], [1, 30, 5] + [0] + [7 * i % 50 for i in range(20)], H, H_kv, D,
                  16, DT[dt])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 256])
def test_shared_page_sizes(dt, page):
    _check_shared([5, 2], [500, 130], [0, 1, 17, 100, 3, 64, 0], 8, 2, 64, page, DT[dt], seed=page,
                  layout="nhd" if page % 2 else "hnd")


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("window", [1, 20, 128, 400, 10000])
def test_shared_window(dt, window):
    _check_shared([4, 3], [300, 1000], [0, 10, 200, 500, 5, 77, 300], 8, 2, 64, 16, DT[dt], window=window,
                  seed=window)


@pytest.mark.parametrize("dt,D", [("bf16", 64), ("f16", 128), ("f32", 64)])
def test_shared_long_prefix(dt, D):
    _check_shared([70, 2], [10000, 20000], [(31 * i) % 200 for i in range(72)], 8, 2, D, 64, DT[dt], seed=3)


def test_shared_without_prefixes_is_decode():
    from dcr_b200.kernel.cuda import paged_attention, paged_shared_attention
    lengths = [33, 0, 512, 100]
    k, v, table = paged_ref.make_pool(lengths, 2, 16, 64, torch.float32, DEV, _gen(21))
    q = torch.randn(4, 8, 64, generator=_gen(22), device=DEV)
    a, la = paged_attention(q, k, v, table, _i32(lengths), return_lse=True)
    b, lb = paged_shared_attention(q, k, v, table, _i32(lengths), _i32([0, 4]), _i32([0] * 4), return_lse=True)
    assert (a - b).abs().max() <= 4 * paged_ref.EPS * a.abs().max() and (b[1] == 0).all()
    assert torch.allclose(la, lb, rtol=0, atol=8 * paged_ref.EPS * 16) and _status() == 0


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_shared_prefixes_that_differ_within_a_group(dt):
    """Members may share less than others, an idle one has length 0, a prefix may pass the length."""
    from dcr_b200.kernel.cuda import paged_shared_attention
    n = 300
    k, v, table1 = paged_ref.make_pool([n, 150], 2, 16, 64, DT[dt], DEV, _gen(23))
    own = table1[1]
    table = torch.stack([table1[0], torch.cat((table1[0, :3], own[:10], own.new_full((6,), -1)))[:19],
                         table1[0], table1[0]])
    lengths, prefix = [n, 3 * 16 + 150, 0, 77], [200, 48, 100, 500]
    q = torch.randn(4, 4, 64, generator=_gen(24), device=DEV).to(DT[dt])
    o, lse = paged_shared_attention(q, k, v, table, _i32(lengths), _i32([0, 4]), _i32(prefix), return_lse=True)
    want = ref.attend(q, k, v, table, [0] * 4, lengths, weight_unit=0.0 if dt == "f32" else 2.0 ** -16)
    _compare(o, lse, want)
    assert _status() == 0


def test_shared_bad_groups_are_reported():
    from dcr_b200.kernel.cuda import paged_shared_attention
    q, k, v, table, lengths, prefix, groups, o = _check_shared([3, 2], [64, 32], [5, 6, 7, 8, 9], 4, 2, 64, 16,
                                                               torch.bfloat16)
    for bad in ([0, 2, 4], [1, 3, 5], [0, 9, 5], [-1, 3, 5], [0, 5, 3]):
        paged_shared_attention(q, k, v, table, _i32(lengths), _i32(bad), _i32(prefix))
        assert _status() != 0, bad
    assert torch.equal(paged_shared_attention(q, k, v, table, _i32(lengths), _i32(groups), _i32(prefix)), o)
    # negative prefixes share nothing
    full = paged_shared_attention(q, k, v, table, _i32(lengths), _i32(groups), _i32([-4] * 5))
    assert (full.float() - o.float()).abs().max() <= 2.0 ** -7 * o.float().abs().max() and _status() == 0


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_shared_captured_twice_in_place_and_streams(dt):
    """Two graphs with a workspace each, replayed in turn, and an eager call between them."""
    from dcr_b200.kernel.cuda import paged_shared_attention
    q, k, v, table, lengths, prefix, groups, o = _check_shared([9, 4], [700, 128], list(range(13)), 8, 2, 64, 16,
                                                               DT[dt], seed=25)
    args = (k, v, table, _i32(lengths), _i32(groups), _i32(prefix))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_shared_attention(q, *args))
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        assert torch.equal(paged_shared_attention(q, *args), o)
    assert torch.equal(outs[0], o) and torch.equal(outs[1], o)
    same = q.clone()
    assert torch.equal(paged_shared_attention(same, *args, out=same), o)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = paged_shared_attention(q, *args)
    side.synchronize()
    assert torch.equal(other, o)


def test_shared_refusals():
    from dcr_b200.kernel.cuda import paged_shared_attention
    q, k, v, table, lengths, prefix, groups, _ = _check_shared([2, 1], [64, 32], [5, 6, 7], 4, 2, 64, 16,
                                                               torch.bfloat16)
    good = dict(q=q, k_pages=k, v_pages=v, page_table=table, lengths=_i32(lengths), groups=_i32(groups),
                prefix=_i32(prefix))
    for bad in (dict(groups=_i32([0])), dict(groups=_i32([0, 1, 1, 2, 3])), dict(groups=_i32([[0, 3]])),
                dict(groups=_i32(groups).long()), dict(prefix=_i32(prefix)[:2]), dict(window=-1),
                dict(q=q[:2]), dict(page_table=table[:2]), dict(out=q[:2])):
        with pytest.raises(AssertionError):
            paged_shared_attention(**dict(good, **bad))
    with pytest.raises(RuntimeError):
        paged_shared_attention(**dict(good, prefix=_i32(prefix).cpu()))


# -------------------------------------------------------------------------------------- rotary
def _frequencies(rot):
    from dcr_b200.kernel.cuda import rotary_frequencies
    return rotary_frequencies(rot, 500000.0, scaling="llama3", factor=8.0, device=DEV)[0]


def _check_turned(got, x, positions, inv, interleaved, factor, **kw):
    want, tol = ref.turn(x, positions, inv, interleaved, factor, x.dtype, **kw)
    d = (got.double() - want).abs()
    assert (d <= tol).all(), float((d / tol).max())


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 64), (64, 32), (64, 16), (64, 2), (80, 80), (80, 20), (128, 96),
                                   (96, 48), (8, 8), (256, 64), (512, 512), (72, 26)])
def test_rotary_layouts(dt, interleaved, D, rot):
    from dcr_b200.kernel.cuda import rotary
    T, g = 37, _gen(D + rot)
    q = torch.randn(T, 6, D, generator=g, device=DEV).to(DT[dt])
    k = torch.randn(T, 2, D, generator=g, device=DEV).to(DT[dt])
    pos, inv = torch.randint(0, 200000, (T,), generator=g, device=DEV).int(), _frequencies(rot)
    a, b = rotary(q, k, inv, pos, interleaved=interleaved, factor=1.25)
    _check_turned(a, q, pos, inv, interleaved, 1.25)
    _check_turned(b, k, pos, inv, interleaved, 1.25)
    # in place, in slices of packed rows: the same bits, and nothing else is touched
    packed = torch.full((T, 11, D), 3.0, device=DEV).to(DT[dt])
    packed[:, 1:7], packed[:, 8:10] = q, k
    x, y = packed[:, 1:7], packed[:, 8:10]
    r = rotary(x, y, inv, pos.long(), interleaved=interleaved, factor=1.25, q_out=x, k_out=y)
    assert r[0].data_ptr() == x.data_ptr() and torch.equal(x, a) and torch.equal(y, b)
    assert (packed[:, 0] == 3).all() and (packed[:, 7] == 3).all() and (packed[:, 10] == 3).all()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("T,H,H_kv", [(1, 1, 1), (1, 32, 8), (3, 5, 1), (1000, 3, 3), (2500, 32, 8)])
def test_rotary_shapes(dt, T, H, H_kv):
    from dcr_b200.kernel.cuda import rotary
    g = _gen(T)
    q = torch.randn(T, H, 64, generator=g, device=DEV).to(DT[dt])
    k = torch.randn(T, H_kv, 64, generator=g, device=DEV).to(DT[dt])
    pos, inv = torch.randint(0, 9000, (T,), generator=g, device=DEV), _frequencies(64)
    a, b = rotary(q, k, inv, pos)
    _check_turned(a, q, pos, inv, False, 1.0)
    _check_turned(b, k, pos, inv, False, 1.0)


@pytest.mark.parametrize("far", [0, -5, 1 << 20, (1 << 31) - 1])
def test_rotary_far_positions(far):
    from dcr_b200.kernel.cuda import rotary
    g = _gen(1)
    x = torch.randn(9, 4, 64, generator=g, device=DEV)
    pos = torch.full((9,), far, dtype=torch.int64, device=DEV) - torch.arange(9, device=DEV)
    inv = _frequencies(64)
    for p in (pos, pos.int()):
        a, _ = rotary(x, x.clone(), inv, p)
        _check_turned(a, x, pos, inv, False, 1.0)


def test_rotary_graph_stream_and_values():
    from dcr_b200.kernel.cuda import rotary
    x = torch.randn(8, 4, 64, device=DEV)
    x[2, 1, 5], x[3, 2, 60] = float("nan"), float("inf")
    pos, inv = torch.arange(8, device=DEV), _frequencies(32)
    a, b = rotary(x, x[:, :1], inv, pos)
    assert torch.equal(a[..., 32:].nan_to_num(9), x[..., 32:].nan_to_num(9))
    assert int(torch.isnan(a).any(-1).sum()) == 1  # a row's NaN stays in it
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c, _ = rotary(x, x[:, :1], inv, pos)
    pos.add_(5)
    graph.replay()
    assert torch.equal(c.nan_to_num(9), rotary(x, x[:, :1], inv, pos)[0].nan_to_num(9))


def test_rotary_refusals():
    from dcr_b200.kernel.cuda import rotary
    x = torch.randn(8, 6, 64, device=DEV)
    q, k, pos, inv = x[:, :4], x[:, 4:], torch.arange(8, device=DEV), _frequencies(64)
    rotary(q, k, inv, pos, q_out=q, k_out=k)
    for args, kw in [((q, k[:7], inv, pos), {}), ((q, k.half(), inv, pos), {}), ((q, k, inv.half(), pos), {}),
                     ((q, k, _frequencies(66), pos), {}), ((q, k, inv, pos.float()), {}),
                     ((q, k, inv, pos[:7]), {}), ((q[..., :6], k[..., :6], inv[:2], pos), {}),
                     ((q.transpose(1, 2), k.transpose(1, 2), inv[:1], pos), {}),
                     ((q, k, inv, pos), dict(q_out=k[:, :1].expand(8, 4, 64))),
                     ((q, k, inv, pos), dict(q_out=x[:, 1:5])), ((q, k, inv, pos), dict(k_out=x[:, 3:5])),
                     ((q, k, inv, pos), dict(k_out=x[:, 2:4], q_out=q)),
                     ((q, k, inv, pos), dict(q_out=torch.empty(8, 4, 64, device=DEV).half()))]:
        with pytest.raises(AssertionError):
            rotary(*args, **kw)
    with pytest.raises(RuntimeError):
        rotary(q, k, inv.cpu(), pos)
    assert rotary(q[:0], k[:0], inv, pos[:0])[0].shape == (0, 4, 64)


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot,norm", [(64, 64, True), (64, 48, False), (64, 20, True), (128, 96, True),
                                        (128, 128, False), (128, 32, True), (128, 6, False)])
def test_rotary_append(dt, interleaved, D, rot, norm):
    from dcr_b200.kernel.cuda import paged_rotary_append
    H, H_kv, page, g = 6, 2, 16, _gen(rot)
    lengths = [40, 1, 100, 16]
    k_pages, v_pages, table = paged_ref.make_pool(lengths, H_kv, page, D, DT[dt], DEV, g)
    seq = [0] * 7 + [1] + [2] * 30 + [3] * 2 + [2]
    slots = list(range(33, 40)) + [0] + list(range(70, 100)) + [15, -1] + [3]
    T = len(seq)
    packed = torch.randn(T, H + 2 * H_kv, D, generator=g, device=DEV).to(DT[dt])
    q, k, v = packed[:, :H], packed[:, H:H + H_kv], packed[:, H + H_kv:]
    w = [(1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(DT[dt]) if norm else None for _ in range(2)]
    pos, inv = torch.randint(0, 100000, (T,), generator=g, device=DEV).int(), _frequencies(rot)
    weights = torch.rand(4, H_kv, table.shape[1] * page, generator=g, device=DEV)
    where = torch.full(weights.shape, -7, dtype=torch.int32, device=DEV)
    before = k_pages.clone(), v_pages.clone(), weights.clone()
    out = paged_rotary_append(q, k, v, inv, pos, k_pages, v_pages, table, _i32(slots), seq=_i32(seq),
                              interleaved=interleaved, factor=1.5, q_weight=w[0], k_weight=w[1], eps=1e-5,
                              weights=weights, pos=where)
    _check_turned(out, q, pos, inv, interleaved, 1.5, weight=w[0])
    held = [i for i, s in enumerate(slots) if s >= 0]
    s, b = _i32(slots)[held].long(), _i32(seq)[held].long()
    pg = table[b, s // page].long()
    _check_turned(k_pages[pg, :, s % page], k[held], pos[held], inv, interleaved, 1.5, weight=w[1])
    assert torch.equal(v_pages[pg, :, s % page], v[held])
    assert (weights[b, :, s] == 0).all() and torch.equal(where[b, :, s], pos[held][:, None].expand(-1, H_kv))
    for now, old in zip((k_pages, v_pages), before):  # nothing else is touched
        now, old = now.clone(), old.clone()
        now[pg, :, s % page] = 0
        old[pg, :, s % page] = 0
        assert torch.equal(now.nan_to_num(9), old.nan_to_num(9))
    assert int((weights != before[2]).sum()) <= len(held) * H_kv and int((where != -7).sum()) == len(held) * H_kv
    assert _status() == 0


def test_rotary_append_matches_tables():
    """Halves of whole heads: paged_append with fp32 tables of the same angles."""
    from dcr_b200.kernel.cuda import paged_append, paged_rotary_append
    g = _gen(31)
    T, D = 50, 64
    q, k, v = (torch.randn(T, h, D, generator=g, device=DEV) for h in (8, 2, 2))
    inv, pos = _frequencies(D), torch.arange(T, device=DEV).int()
    angle = torch.arange(T, device=DEV).double()[:, None] * inv.double()
    angle = torch.cat((angle, angle), 1)
    pools = [[torch.zeros(4, 2, 16, D, device=DEV) for _ in range(2)] for _ in range(2)]
    table, seq = _i32([[2, 0, 1, 3]]), torch.zeros(T, dtype=torch.int32, device=DEV)
    a = paged_append(q, k, v, angle.cos().float(), angle.sin().float(), pos, *pools[0], table, pos, seq=seq)
    b = paged_rotary_append(q, k, v, inv, pos, *pools[1], table, pos, seq=seq)
    # both within 2^-22 + some roundings of the definition, for sums of two products
    assert (a - b).abs().max() <= 2.0 ** -20 * q.abs().max()
    assert (pools[0][0] - pools[1][0]).abs().max() <= 2.0 ** -20 * k.abs().max()
    assert torch.equal(pools[0][1], pools[1][1])


def test_rotary_append_bad_places_and_refusals():
    from dcr_b200.kernel.cuda import paged_rotary_append
    q, k, v = (torch.randn(2, h, 64, device=DEV) for h in (4, 2, 2))
    kp, vp = torch.zeros(2, 2, 16, 64, device=DEV), torch.zeros(2, 2, 16, 64, device=DEV)
    table, inv, pos = _i32([[0, -1], [1, 9]]), _frequencies(64), _i32([3, 4])
    good = dict(q=q, k=k, v=v, inv_freq=inv, positions=pos, k_pages=kp, v_pages=vp, page_table=table,
                slots=_i32([1, 2]))
    paged_rotary_append(**good)
    assert _status() == 0
    for slots, seq in (([40, 2], None), ([17, 2], None), ([1, 20], None), ([1, 2], [0, 2]), ([1, 2], [-1, 1])):
        paged_rotary_append(**dict(good, slots=_i32(slots), seq=None if seq is None else _i32(seq)))
        assert _status() != 0
    for bad in (dict(inv_freq=_frequencies(128)), dict(positions=pos.long()), dict(q=q[:, :3]),
                dict(slots=_i32([1])), dict(q_weight=inv), dict(weights=torch.zeros(2, 2, 5, device=DEV)),
                dict(k=k.half()), dict(out=q[:1])):
        with pytest.raises(AssertionError):
            paged_rotary_append(**dict(good, **bad))
    three = {n: torch.cat((good[n], good[n][:1])) for n in ("q", "k", "v", "positions", "slots")}
    with pytest.raises(AssertionError):
        paged_rotary_append(**dict(good, **three))  # three tokens, two sequences


# ---------------------------------------------------------------------------- all of them, as in use
@pytest.mark.parametrize("dt", sorted(DT))
def test_prompts_forks_and_steps_together(dt):
    """A prompt in two chunks, its pages shared by three continuations, two decode steps: every token's
    attention against one contiguous definition."""
    from dcr_b200.kernel.cuda import paged_prefill, paged_rotary_append, paged_shared_attention
    H, H_kv, D, page, g = 8, 2, 64, 16, _gen(41)
    inv, P, B = _frequencies(32), 96, 3
    kp, vp = (torch.full((20, H_kv, page, D), float("nan"), device=DEV).to(DT[dt]) for _ in "kv")
    table = torch.full((B, 8), -1, dtype=torch.int32, device=DEV)
    table[:, :6] = torch.arange(6, device=DEV).int() + 3
    table[:, 6] = torch.arange(B, device=DEV).int() + 12
    unit = 0.0 if dt == "f32" else paged_ref.UNIT[DT[dt]]

    def rows(T):
        return [torch.randn(T, h, D, generator=g, device=DEV).to(DT[dt]) for h in (H, H_kv, H_kv)]

    for a, b in ((0, 50), (50, P)):
        q, k, v = rows(b - a)
        at = torch.arange(a, b, device=DEV).int()
        q = paged_rotary_append(q, k, v, inv, at, kp, vp, table[:1], at, seq=torch.zeros_like(at), interleaved=True)
        o, lse = paged_prefill(q, kp, vp, table[:1], _i32([b]), _i32([0, b - a]), return_lse=True)
        lo, hi, seq = ref.prefill_limits([0, b - a], [b], 0, True)
        _compare(o, lse, ref.attend(q, kp, vp, table[seq], lo, hi, weight_unit=unit))
    for step in range(2):
        q, k, v = rows(B)
        at = torch.full((B,), P + step, dtype=torch.int32, device=DEV)
        q = paged_rotary_append(q, k, v, inv, at, kp, vp, table, at, interleaved=True)
        n = [P + step + 1] * B
        o, lse = paged_shared_attention(q, kp, vp, table, _i32(n), _i32([0, B]), _i32([P] * B), return_lse=True)
        _compare(o, lse, ref.attend(q, kp, vp, table, [0] * B, n,
                                    weight_unit=0.0 if dt == "f32" else 2.0 ** -16))
    assert _status() == 0
