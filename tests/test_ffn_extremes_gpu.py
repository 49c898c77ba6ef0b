"""Gradients of the feed-forward operators where their factors leave the range: infinities
behind an inactive unit, arguments whose powers fp32 does not hold, products beyond fp16."""
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


def test_half_precision_range():
    """The products' gradients are rounded to the operands' type on the way to A's and B's:
    in fp16 one beyond 65504 is infinite, and so is what it goes into, never a finite value
    that is wrong."""
    def step(dtype, gate, up, dh):
        x = torch.full((1, 1), 4.0, dtype=dtype, device="cuda", requires_grad=True)
        g, u = (torch.full((1, 1), v, dtype=dtype, device="cuda", requires_grad=True)
                for v in (gate, up))
        h = bg.matmul_b200_gated(x, g, u, activation="none")
        return [float(t) for t in torch.autograd.grad(h, (x, g, u), torch.full_like(h, dh))]
    # dz = (dh u, dh g); dx = dz . (gate, up), dgate = dz[0] x, dup = dz[1] x.  All exact.
    for dtype in (torch.float16, torch.bfloat16):
        assert step(dtype, 1.0, 0.25, 2048.0) == [4096.0, 8192.0, 32768.0]
    # dz = (1, 307200): past fp16's range, where dx = 300 + 300 is not
    assert step(torch.bfloat16, 300.0, 2.0 ** -10, 256.0) == [600.0, 4.0, 1228800.0]
    assert step(torch.float16, 300.0, 2.0 ** -10, 256.0) == [math.inf, 4.0, math.inf]


def test_clipping_at_its_borders():
    """The factor is min(1, max_norm / (norm + 1e-6)), also where the norm is of the size of
    that 1e-6 and where both are infinite (it is then NaN)."""
    g = torch.tensor([4e-7, 0.0], device="cuda")
    norm = bg.clip_grads_b200([g], 5e-7)
    want = 4e-7 * 5e-7 / (4e-7 + 1e-6)
    # (norm, factor and product rounded once each, the input twice: 2^-21 holds them)
    assert abs(float(norm) - 4e-7) <= 2.0 ** -21 * 4e-7
    assert abs(float(g[0]) - want) <= 2.0 ** -21 * want and float(g[1]) == 0.0
    g = torch.tensor([2.0, math.inf], device="cuda")
    assert float(bg.clip_grads_b200([g], math.inf)) == math.inf and bool(g.isnan().all())
    g = torch.tensor([2.0, 3e38, -3e38], device="cuda")   # a norm beyond fp32, not beyond fp64
    keep = g.clone()
    assert float(bg.clip_grads_b200([g], math.inf)) == math.inf and torch.equal(g, keep)
