"""Shared prefixes where some sequences of a group wait (a length of 0) or share less than the others: the
same results, and a prefix that is still dealt to all SMs."""
from __future__ import annotations

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import rows_ref as ref  # noqa: E402
from test_gpu_prompts import DEV, DT, _compare, _gen, _i32, _make_shared, _status  # noqa: E402

pytestmark = pytest.mark.gpu


def _time(f, calls=10):
    """Microseconds of a call among others, the least of several runs of a captured graph."""
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(calls):
            f()
    best = float("inf")
    for _ in range(8):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 1000 / calls)
    return best


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("change", ["waits", "shares little", "shares nothing"])
def test_a_group_whose_first_sequence_sees_little_is_cut_up(dt, change):
    """With the first sequence's slots as the measure one CTA a KV head walked the whole prefix: 256 tiles one
    after another instead of about 18, 10 to 24 times the time. Three times is far from both."""
    from dcr_b200.kernel.cuda import paged_shared_attention
    k, v, table, n, prefix, groups = _make_shared([8], [32768], [64] * 8, 8, 16, 64, DT[dt], 1)
    q = torch.randn(8, 16, 64, generator=_gen(2), device=DEV).to(DT[dt])

    def time_of(n, prefix):
        args = (q, k, v, table, _i32(n), _i32(groups), _i32(prefix))
        return _time(lambda: paged_shared_attention(*args))
    whole = time_of(n, prefix)
    less = time_of(*((([0] + n[1:]), prefix) if change == "waits" else
                     (n, [16 if change == "shares little" else 0] + prefix[1:])))
    assert less <= 3 * whole and _status() == 0


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("idle", [0, 7])
def test_a_sequence_that_waits_leaves_whole_tiles_whole(dt, idle):
    """With its row among the limits no tile of the prefix came by tensor-map copies, and each was masked and
    searched for values that are not finite: twice the time. 1.4 is halfway on a logarithm."""
    from dcr_b200.kernel.cuda import paged_shared_attention
    k, v, table, n, prefix, groups = _make_shared([16], [32768], [64] * 16, 8, 32, 128, DT[dt], 1)
    q = torch.randn(16, 64, 128, generator=_gen(2), device=DEV).to(DT[dt])

    def time_of(n):
        args = (q, k, v, table, _i32(n), _i32(groups), _i32(prefix))
        return _time(lambda: paged_shared_attention(*args))
    assert time_of([0 if b == idle else x for b, x in enumerate(n)]) <= 1.4 * time_of(n) and _status() == 0


def _check_idle(members, prefixes, owns, idle, H, H_kv, page, D, dt, *, window=0, seed=0, spoil=None):
    """Some sequences wait; a value or key in the prefix that is not finite spoils none of them."""
    from dcr_b200.kernel.cuda import paged_shared_attention
    k, v, table, n, prefix, groups = _make_shared(members, prefixes, owns, H_kv, page, D, dt, seed)
    n = [0 if b in idle else x for b, x in enumerate(n)]
    q = torch.randn(len(n), H, D, generator=_gen(seed + 1), device=DEV).to(dt)
    for b in idle:
        q[b] = float("nan") if spoil else 1e4
    spoilt = torch.zeros(q.shape[:2], dtype=torch.bool, device=DEV)
    if spoil:
        # a slot in the middle of the first group's prefix, which the others all see
        at = prefix[0] // 2
        v[table[0, at // page].long(), 0, at % page, 5] = spoil
        spoilt[[b for b in range(groups[1]) if b not in idle], :H // H_kv] = True
    o, lse = paged_shared_attention(q, k, v, table, _i32(n), _i32(groups), _i32(prefix), window=window,
                                    return_lse=True)
    assert all((o[b] == 0).all() and (lse[b] == float("-inf")).all() for b in idle)
    assert torch.isfinite(o[~spoilt]).all() and not torch.isfinite(o[spoilt][:, 5]).any()
    lo = [max(0, x - window) if window else 0 for x in n]
    want = ref.attend(torch.nan_to_num(q, nan=0.0), k, v, table, lo, n,
                      weight_unit=0.0 if dt == torch.float32 else 2.0 ** -16)
    want[0][spoilt] = 0
    _compare(torch.where(spoilt[..., None], 0, o).to(dt), lse, want)
    assert _status() == 0


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("idle", [(0,), (3,), (0, 1, 2), (5, 6), (0, 1, 2, 3, 4, 5, 6)])
@pytest.mark.parametrize("window", [0, 300])
def test_sequences_that_wait(dt, idle, window):
    _check_idle([4, 3], [640, 300], [5, 9, 3, 1, 8, 70, 4], idle, 8, 2, 16, 64, DT[dt], window=window, seed=3)


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("D,G", [(64, 4), (128, 16), (64, 16)])
@pytest.mark.parametrize("spoil", [None, float("inf"), float("nan")])
def test_sequences_that_wait_in_a_large_group(dt, D, G, spoil):
    """More rows than one block, with rows that wait in every warp, before and behind those that do not."""
    idle = [b for b in range(24) if b % 3 == 0 or b > 20]
    _check_idle([24], [2000], [1 + b for b in range(24)], idle, 2 * G, 2, 16, D, DT[dt], seed=4, spoil=spoil)


def test_more_groups_than_weights_are_kept_of():
    """Groups of one, most of which wait."""
    B = 700
    _check_idle([1] * B, [48] * B, [3] * B, [b for b in range(B) if b % 7], 1, 1, 16, 64, torch.bfloat16, seed=5)


@pytest.mark.parametrize("dt,groups,D", [("bf16", 24, 64), ("f16", 40, 128), ("bf16", 70, 64), ("f32", 80, 64)])
@pytest.mark.parametrize("window", [0, 200])
def test_more_units_than_are_cut_up(dt, groups, D, window):
    """Groups times KV heads past the SMs (four times past them in fp32): a CTA a unit, a place a row; up to 64
    groups by what they see, more in their order."""
    members = [1 + g % 3 for g in range(groups)]
    B = sum(members)
    idle = [b for b in range(B) if b % 11 == 4]
    _check_idle(members, [16 * (1 + g * 7 % 30) for g in range(groups)], [1 + b % 40 for b in range(B)], idle, 16, 8,
                16, D, DT[dt], window=window, seed=6)
