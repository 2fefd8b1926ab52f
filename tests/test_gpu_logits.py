"""Penalties, bias, mask and greedy token on the GPU against the definition in 64 bits."""
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


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _first_largest(x, ok):
    """The lowest index of the largest value (NaN above all) among the allowed, -1 without one."""
    i = torch.nonzero(ok).flatten()
    if not len(i):
        return -1
    y = x[i].double()
    nan = torch.nonzero(y.isnan()).flatten()
    return int(i[nan[0]] if len(nan) else i[torch.nonzero(y == y.max()).flatten()[0]])


def _check(B, V, L, dt, *, bias=None, mask=None, wide=0, tok=torch.int32, seed=0, spread=None):
    from dcr_b200.kernel.cuda.logits import process_logits
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(B, V + wide, generator=g, device=DEV).mul(4).to(DT[dt])[:, :V]
    tokens = torch.randint(0, spread or V, (B, L), generator=g, device=DEV).to(tok)
    if L > 3:
        tokens[:, 2] = -1  # padding
    n = [(L * (b + 1)) // B if b else 0 for b in range(B)] if B > 1 else [L]
    prompt = [m // 2 if b % 3 else m + 5 for b, m in enumerate(n)]  # the whole of it, too
    rep, pres, freq = (lo + torch.rand(B, generator=g, device=DEV) for lo in (0.9, -0.5, 0.0))
    bs = None
    if bias is not None:
        bs = torch.randn(*((V,) if bias == "one" else (B, V)), generator=g, device=DEV)
    al = None
    if mask is not None:
        al = torch.randint(-2**31, 2**31, (B, (V + 31) // 32), generator=g, device=DEV).to(torch.int32)
        if mask == "none":
            al.zero_()
        elif V % 32:
            al[:, -1] |= -(1 << (V % 32))  # bits past the vocabulary mean nothing
    y, token = process_logits(x, tokens=tokens if L else None, token_lengths=_i32(n) if L else None,
                              prompt_lengths=_i32(prompt) if L else None, repetition=rep,
                              presence=pres, frequency=freq, bias=bs, allowed=al)
    assert y.dtype == x.dtype and token.dtype == torch.int64
    for b in range(B):
        Y, tol, ok = ref.logits(x[b], tokens[b].tolist(), n[b] if L else 0, min(prompt[b], n[b]) if L else 0,
                                float(rep[b]), float(pres[b]), float(freq[b]),
                                None if bs is None else bs if bs.dim() == 1 else bs[b],
                                None if al is None else al[b])
        assert (y[b][~ok] == -math.inf).all()
        assert ((y[b].double() - Y).abs()[ok] <= tol[ok]).all()
        assert int(token[b]) == _first_largest(y[b], ok)
    from dcr_b200 import _lib
    assert _lib.read_device_status(clear=True) == 0


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("B,V,L", [(1, 1, 1), (1, 31, 0), (3, 1000, 50), (2, 32000, 5000),
                                   (5, 128256, 1000), (1, 128257, 3), (4, 4099, 20000)])
@pytest.mark.parametrize("bias,mask", [(None, None), ("one", "some"), ("each", None), (None, "some")])
def test_process_logits(dt, B, V, L, bias, mask):
    _check(B, V, L, dt, bias=bias, mask=mask)


@pytest.mark.parametrize("dt", sorted(DT))
def test_strided_rows_int64_history_and_empty_masks(dt):
    _check(4, 1001, 300, dt, wide=7, tok=torch.int64, mask="some", bias="each")
    _check(3, 500, 10, dt, mask="none")
    _check(2, 700, 3000, dt, spread=3)  # the same three tokens again and again


@pytest.mark.parametrize("V", [300000, 700001])
def test_large_vocabularies(V):
    _check(2, V, 2000, "bf16", bias="one", mask="some")


def test_history_longer_than_the_tables():
    """The vocabulary is taken in chunks where the counts of a whole slice would not fit."""
    _check(2, 200001, 40000, "f32", bias="one", mask="some")
    _check(1, 3000, 70000, "bf16", tok=torch.int64)


def test_many_rows():
    _check(200, 3001, 64, "bf16", mask="some")


@pytest.mark.parametrize("dt", sorted(DT))
def test_ties_nan_and_infinities(dt):
    from dcr_b200.kernel.cuda.logits import process_logits
    x = torch.zeros(6, 5000, device=DEV).to(DT[dt])
    x[0, 1000:] = 2
    x[1] = -math.inf
    x[2, 77], x[2, 4000] = math.inf, math.inf
    x[3, 4000], x[3, 4500] = math.nan, math.nan
    x[4, :40], x[4, 3000] = -0.0, 0.0
    x[5] = torch.finfo(DT[dt]).min
    ok = torch.full((6, 157), -1, dtype=torch.int32, device=DEV)
    y, t = process_logits(x, allowed=ok)
    assert t.tolist() == [1000, 0, 77, 4000, 0, 0]
    assert torch.equal(y.nan_to_num(3), x.nan_to_num(3))
    ok[:, 0] = 0          # tokens 0..31 are not allowed
    ok[3, 4000 // 32] = 0  # nor is one of the NaN
    x[:, :32] = math.nan
    y, t = process_logits(x, allowed=ok)
    assert t.tolist() == [1000, 32, 77, 4500, 32, 32]
    assert (y[:, :32] == -math.inf).all()


def test_in_place_on_a_stream_and_history_out_of_range():
    from dcr_b200 import _lib
    from dcr_b200.kernel.cuda.logits import process_logits
    x = torch.randn(3, 999, device=DEV)
    tokens = torch.randint(0, 999, (3, 40), device=DEV)
    rep = torch.full((3,), 1.3, device=DEV)
    want, t0 = process_logits(x, tokens=tokens, repetition=rep)
    assert _lib.read_device_status(clear=True) == 0
    wrong = tokens.clone()
    wrong[1, :20] = 999
    process_logits(x, tokens=wrong, repetition=rep)
    assert _lib.read_device_status(clear=True) == _lib.DCR_ERR_DEVICE_INDEX
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y, t = process_logits(x, tokens=tokens, repetition=rep, out=x)
        s.synchronize()
    assert y is x and torch.equal(y, want) and torch.equal(t, t0)


def test_no_rows_and_refusals():
    from dcr_b200.kernel.cuda.logits import process_logits
    x = torch.randn(2, 100, device=DEV)
    y, t = process_logits(x[:0])
    assert y.shape == (0, 100) and t.shape == (0,)
    tok = torch.zeros(2, 4, dtype=torch.int64, device=DEV)
    one = torch.ones(2, device=DEV)
    for kw in (dict(tokens=tok.float()), dict(tokens=tok[:1]), dict(token_lengths=_i32([1, 1])),
               dict(tokens=tok, token_lengths=_i32([1])), dict(repetition=one.double()), dict(presence=one[:1]),
               dict(bias=torch.ones(99, device=DEV)), dict(bias=torch.ones(2, 100, device=DEV).half()),
               dict(allowed=_i32([[1, 2, 3]] * 2)), dict(allowed=torch.ones(2, 4, device=DEV)),
               dict(out=torch.empty(2, 99, device=DEV)), dict(out=x.double())):
        with pytest.raises(AssertionError):
            process_logits(x, **kw)
    with pytest.raises(AssertionError):
        process_logits(x.t())
    with pytest.raises(AssertionError):
        process_logits(x.double())
    with pytest.raises(RuntimeError):
        process_logits(x.cpu())
