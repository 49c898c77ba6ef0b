"""Gradients of the feed-forward operators where their factors leave the range: infinities
behind an inactive unit."""
import math

import pytest
import torch

import blackwell_gemm_b200 as bg

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
