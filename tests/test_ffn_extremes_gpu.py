"""Gradients of the feed-forward operators where their factors leave the range: infinities
behind an inactive unit, arguments whose powers fp32 does not hold."""
import math

import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi
from test_gated_gpu import curve

pytestmark = pytest.mark.gpu


def column(values, dtype=torch.bfloat16):
    return torch.tensor(values, dtype=dtype, device="cuda")[:, None]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_inactive_units_pass_nothing_back(dtype):
    """relu: where its argument is not above zero nothing comes back, whatever arrives."""
    bad = [math.inf, -math.inf, math.nan, math.inf, 2.0, 3.0]
    z = column([-2.0, -1.0, -0.5, 0.0, 3.0, -3.0], dtype)
    dy, one = column(bad, dtype), torch.ones(1, 1, dtype=dtype, device="cuda")
    x, w = z.clone().requires_grad_(), one.clone().requires_grad_()
    b = torch.zeros(1, dtype=dtype, device="cuda", requires_grad=True)
    y = bg.matmul_b200_act(x, w.t(), b, activation="relu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert dx.flatten().tolist() == [0.0, 0.0, 0.0, 0.0, 2.0, 0.0]
    assert float(dw) == 6.0 and float(db) == 2.0
    # (the gate's gradient; the other factor's is act(g) times what arrives)
    h = bg.matmul_b200_gated(z, w.t(), one.t(), activation="relu")
    dgate, = torch.autograd.grad(h, w, dy)
    assert float(dgate) == 18.0   # dh u act'(g) x = 2 * 3 * 1 * 3


@pytest.mark.parametrize("act", capi.ACTIVATIONS)
def test_far_arguments(act):
    """|z| up to the largest bf16 value: act(z) and its slope are those of the limit, to the
    last bit (z, 0 or 1; 1 or 0)."""
    top = float(torch.finfo(torch.bfloat16).max)
    far = [1e9, 2.0 ** 62, 2.0 ** 66, 1e20, 1e30, top]
    x = column([*far, *(-v for v in far)]).requires_grad_()
    one = torch.ones(1, 1, dtype=torch.bfloat16, device="cuda")
    y = bg.matmul_b200_act(x, one, activation=act)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    a, slope = curve(act, x.detach().double())
    assert torch.equal(y.double(), a) and torch.equal(dx.double(), slope)
    h = bg.matmul_b200_gated(one, gate := x.detach().clone().requires_grad_().t(),
                             torch.ones_like(gate), activation=act)
    dgate, = torch.autograd.grad(h, gate, torch.ones_like(h))
    assert torch.equal(h.double(), a.t()) and torch.equal(dgate.double(), slope.t())
