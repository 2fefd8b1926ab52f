"""Outputs of the appends that reach into the keys and values beside them are refused, and nothing is
appended then."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _call(func, packed, out):
    """The append with 2 query heads on 2 KV heads, from rows [T, 6, D]; the pages."""
    T = packed.shape[0]
    pools = torch.zeros(2, 2, 2, 16, 64, device=DEV)
    at = torch.arange(T, device=DEV).int()
    turn = ((torch.ones(32, device=DEV),) if func.__name__ == "paged_rotary_append" else
            (torch.ones(T, 64, device=DEV), torch.zeros(T, 64, device=DEV)))
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV)
    func(packed[:, :2], packed[:, 2:4], packed[:, 4:], *turn, at, pools[0], pools[1], table, at,
         seq=torch.zeros_like(at), out=out)
    return pools


def _refused(func):
    x = torch.randn(3, 6, 64, device=DEV)
    before = x.clone()
    for packed, out in ((x, x.view(9, 2, 64)[:3]), (x, x.view(9, 2, 64)[6:]), (x[:1], x[:1, 2:4]), (x[:1], x[:1, 4:]),
                        (x[:1], x.view(18, 64)[3:5].view(1, 2, 64))):
        with pytest.raises(AssertionError):
            _call(func, packed, out)
    assert torch.equal(x, before)
    whole = torch.empty(3, 2, 64, device=DEV)
    assert (_call(func, x, whole)[1, 1, :, :3] == x[:, 4:].transpose(0, 1)).all()
    assert torch.equal(_call(func, x[:1].clone(), whole[:1])[1, 1, :, :1], x[:1, 4:].transpose(0, 1))
    one = x[:1].clone()
    assert (_call(func, one, one[:, :2])[1, 1, :, :1] == x[:1, 4:].transpose(0, 1)).all()  # the queries themselves


def test_rotary_append():
    from dcr_b200.kernel.cuda import paged_rotary_append
    _refused(paged_rotary_append)


def test_append():
    from dcr_b200.kernel.cuda import paged_append
    _refused(paged_append)
