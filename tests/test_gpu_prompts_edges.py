"""Prompts, shared prefixes and rotations on the GPU: calls that the documentation allows and that are easily
forgotten."""
from __future__ import annotations

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_ref  # noqa: E402
import rows_ref as ref  # noqa: E402
from test_gpu_prompts import (DEV, DT, _check_prefill, _check_shared, _check_turned, _compare, _frequencies,  # noqa: E402
                              _gen, _i32, _status)

pytestmark = pytest.mark.gpu


def _unit(dt):
    return 0.0 if dt == "f32" else paged_ref.UNIT[DT[dt]]


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-3, 3.0])
@pytest.mark.parametrize("news", [[300, 3], [5, 9]])  # two blocks of rows a CTA, or one
def test_prefill_scales(dt, scale, news):
    _check_prefill(news, [400, 200], 4, 1, 64, 16, DT[dt], scale=scale)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_shared_scales(dt, scale):
    _check_shared([4, 2], [300, 64], [3, 9, 20, 0, 5, 6], 8, 2, 64, 16, DT[dt], scale=scale)


@pytest.mark.parametrize("dt,D", [("bf16", 64), ("f16", 128), ("f32", 64)])
def test_shared_as_many_parts_as_there_can_be(dt, D):
    _check_shared([3], [30000], [1, 100, 77], 4, 1, D, 16, DT[dt], seed=5)


@pytest.mark.parametrize("dt", sorted(DT))
def test_prefill_in_parts_in_place(dt):
    """Few rows on a long history are cut into parts; O may still be q itself."""
    from dcr_b200.kernel.cuda import paged_prefill
    q, k, v, table, o, lse = _check_prefill([7, 2], [9000, 4000], 4, 2, 64, 16, DT[dt], seed=6)
    same = q.clone()
    got = paged_prefill(same, k, v, table, _i32([9000, 4000]), _i32([0, 7, 9]), out=same)
    assert got.data_ptr() == same.data_ptr() and torch.equal(same, o)


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("n", [40, 400])
def test_a_query_that_is_not_finite_keeps_to_itself(dt, n):
    from dcr_b200.kernel.cuda import paged_prefill
    k, v, table = paged_ref.make_pool([n], 2, 16, 64, DT[dt], DEV, _gen(7))
    q = torch.randn(n, 4, 64, generator=_gen(8), device=DEV).to(DT[dt])
    q[n // 2, 1, 5], q[3, 2, 0] = float("nan"), float("inf")
    o = paged_prefill(q, k, v, table, _i32([n]), _i32([0, n]))
    bad = torch.zeros(n, 4, dtype=torch.bool, device=DEV)
    bad[n // 2, 1] = bad[3, 2] = True
    assert torch.isfinite(o[~bad]).all() and torch.isnan(o[n // 2, 1]).all()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_calls_on_two_streams_at_once(dt):
    from dcr_b200.kernel.cuda import paged_prefill, paged_shared_attention
    q, k, v, table, o, _ = _check_prefill([600, 300], [900, 2000], 8, 2, 64, 16, DT[dt], seed=9)
    sq, sk, sv, st, n, prefix, groups, so = _check_shared([20, 4], [3000, 500], list(range(24)), 8, 2, 64, 16, DT[dt],
                                                          seed=10)
    args = (k, v, table, _i32([900, 2000]), _i32([0, 600, 900]))
    shared = (sk, sv, st, _i32(n), _i32(groups), _i32(prefix))
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(paged_prefill(q, *args) if i == 0 else paged_shared_attention(sq, *shared))
    torch.cuda.synchronize()
    assert all(torch.equal(x, o) for x in outs[0]) and all(torch.equal(x, so) for x in outs[1])
    assert _status() == 0


def test_one_workspace_for_calls_of_a_stream():
    """Calls that follow one another may share a workspace, two graphs of them too."""
    from dcr_b200.kernel.cuda import paged_shared_attention, paged_shared_workspace_bytes
    calls = []
    ws = torch.empty(max(paged_shared_workspace_bytes(b, 1, 8, 2, 64) for b in (9, 30)), dtype=torch.uint8,
                     device=DEV)
    for b in (9, 30):
        q, k, v, table, n, prefix, groups, o = _check_shared([b], [2000], list(range(b)), 8, 2, 64, 16,
                                                             torch.bfloat16, seed=b)
        args = (q, k, v, table, _i32(n), _i32(groups), _i32(prefix))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = paged_shared_attention(*args, workspace_buf=ws)
        calls.append((graph, out, o))
    for _ in range(5):
        for graph, _, _ in calls:
            graph.replay()
    torch.cuda.synchronize()
    for _, out, o in calls:
        assert torch.equal(out, o)


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("rot,norm", [(64, True), (20, True), (32, False)])
def test_rotary_append_into_the_queries(dt, rot, norm):
    from dcr_b200.kernel.cuda import paged_rotary_append
    g, T, D = _gen(11), 9, 64
    q, k, v = (torch.randn(T, h, D, generator=g, device=DEV).to(DT[dt]) for h in (4, 2, 2))
    w = (1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(DT[dt]) if norm else None
    pools = torch.zeros(2, 3, 2, 16, D, device=DEV).to(DT[dt])
    pos, inv = torch.arange(T, device=DEV).int(), _frequencies(rot)
    same = q.clone()
    got = paged_rotary_append(same, k, v, inv, pos, pools[0], pools[1], _i32([[2, 0]]), pos,
                              seq=torch.zeros_like(pos), q_weight=w, k_weight=w, out=same)
    assert got.data_ptr() == same.data_ptr()
    _check_turned(same, q, pos, inv, False, 1.0, weight=w)


def test_rotary_of_broadcast_rows():
    """Inputs may be expanded; outputs are rows of their own."""
    from dcr_b200.kernel.cuda import rotary
    x = torch.randn(1, 1, 64, device=DEV).expand(7, 3, 64)
    pos, inv = torch.arange(7, device=DEV), _frequencies(64)
    a, b = rotary(x, x, inv, pos)
    _check_turned(a, x, pos, inv, False, 1.0)
    assert torch.equal(a, b)
    with pytest.raises(AssertionError):
        rotary(x, x.contiguous(), inv, pos, q_out=x)


def test_prefill_of_more_sequences_than_are_sorted():
    for B in (64, 65, 200):
        news = [1 + (7 * b) % 5 for b in range(B)]
        _check_prefill(news, [n + (53 * b) % 300 for b, n in enumerate(news)], 8, 4, 64, 16, torch.float16, seed=B)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_prefill_lengths_of_one(dt):
    _check_prefill([1] * 5, [1] * 5, 16, 1, 128, 1, DT[dt])


def test_prefill_pool_of_other_strides():
    """A pool that is a slice of a larger one, its heads and slots apart by more than their rows."""
    from dcr_b200.kernel.cuda import paged_prefill
    q, k, v, table, o, _ = _check_prefill([150, 20], [300, 20], 8, 2, 64, 16, torch.bfloat16, seed=12)
    wide = torch.full((k.shape[0] + 2, 16, 5, 3, 64), float("nan"), dtype=torch.bfloat16, device=DEV)
    ks, vs = wide[1:-1, :, 1:5:2, 0].transpose(1, 2), wide[1:-1, :, 1:5:2, 2].transpose(1, 2)
    ks.copy_(k), vs.copy_(v)
    assert torch.equal(paged_prefill(q, ks, vs, table, _i32([300, 20]), _i32([0, 150, 170])), o)
    lo, hi, seq = ref.prefill_limits([0, 150, 170], [300, 20], 0, True)
    got, lse = paged_prefill(q, ks, vs, table, _i32([300, 20]), _i32([0, 150, 170]), return_lse=True)
    _compare(got, lse, ref.attend(q, k, v, table[seq], lo, hi, weight_unit=_unit("bf16")))
