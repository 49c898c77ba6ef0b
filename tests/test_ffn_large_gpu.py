"""Feed-forward operators past 2^31 elements: rows and features picked from the far end against
64 bits.  (Tolerances as in test_gated_gpu.py, of the same formulas.)"""
import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi
from test_gated_gpu import BEND, E, curve, within

pytestmark = pytest.mark.gpu

U = 2.0 ** -8


@pytest.fixture(autouse=True)
def _clean():
    capi.device_status(True)
    torch.cuda.empty_cache()
    yield
    assert capi.device_status(True) == 0
    torch.cuda.empty_cache()


def test_gated_step():
    m, n, k = 66000, 33000, 64     # 2.2e9 elements of h, twice that of the kept products
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(m, k, generator=g, device="cuda").bfloat16().requires_grad_()
    wg, wu = ((torch.randn(n, k, generator=g, device="cuda") / 8).bfloat16().requires_grad_()
              for _ in range(2))
    dh = torch.randn(m, n, generator=g, device="cuda", dtype=torch.bfloat16)
    h = bg.matmul_b200_gated(x, wg.t(), wu.t())
    dx, dwg, dwu = torch.autograd.grad(h, (x, wg, wu), dh)
    xd, gd, ud = (t.detach().double() for t in (x, wg, wu))

    def parts(rows, cols):
        d = dh[rows][:, cols].double()
        gs, us = xd[rows] @ gd[cols].T, xd[rows] @ ud[cols].T
        eg, eu = (E * (k + 1) * (xd[rows].abs() @ w[cols].abs().T) for w in (gd, ud))
        y, slope = curve("silu", gs)
        return d, gs, us, eg, eu, y, slope
    everything = slice(None)
    rows = torch.tensor([0, 1, 40000, 65023, 65999], device="cuda")
    d, gs, us, eg, eu, y, slope = parts(rows, everything)
    within(h[rows], y * us, U * (y * us).abs() + (BEND * eg + 2.0 ** -18 * y.abs()) * us.abs()
           + y.abs() * eu + BEND * eg * eu, "h")
    dg, du = d * us * slope, d * y
    fg = (U + 2.0 ** -17) * dg.abs() + d.abs() * BEND * (eu + us.abs() * eg + eu * eg) \
        + d.abs() * us.abs() * 2.0 ** -20
    fu = (U + 2.0 ** -17) * du.abs() + d.abs() * BEND * eg + d.abs() * 2.0 ** -20 * y.abs()
    want = dg @ gd + du @ ud
    within(dx[rows], want, U * want.abs() + fg @ gd.abs() + fu @ ud.abs()
           + E * 2 * (n + 1) * (dg.abs() @ gd.abs() + du.abs() @ ud.abs()), "dx")
    cols = torch.tensor([0, 16500, 32999], device="cuda")
    d, gs, us, eg, eu, y, slope = parts(everything, cols)
    dg, du = d * us * slope, d * y
    fg = (U + 2.0 ** -17) * dg.abs() + d.abs() * BEND * (eu + us.abs() * eg + eu * eg) \
        + d.abs() * us.abs() * 2.0 ** -20
    fu = (U + 2.0 ** -17) * du.abs() + d.abs() * BEND * eg + d.abs() * 2.0 ** -20 * y.abs()
    for got, a, f in ((dwg[cols], dg, fg), (dwu[cols], du, fu)):
        want = a.T @ xd
        within(got, want, U * want.abs() + f.T @ xd.abs() + E * (m + 1) * (a.abs().T @ xd.abs()), "dw")


def test_act_with_residual():
    m, n, k = 66000, 33000, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    w = (torch.randn(n, k, generator=g, device="cuda") / 8).bfloat16()
    b = torch.randn(n, generator=g, device="cuda").bfloat16()
    r = torch.randn(m, n, generator=g, device="cuda", dtype=torch.bfloat16)
    y = bg.matmul_b200_act(x, w.t(), b, r, activation="gelu")
    rows = torch.tensor([0, 33333, 65999], device="cuda")
    z = x[rows].double() @ w.double().T + b.double()
    ez = E * (k + 2) * (x[rows].double().abs() @ w.double().abs().T + b.double().abs())
    a, _ = curve("gelu", z)
    want = a + r[rows].double()
    within(y[rows], want, U * want.abs() + BEND * ez + 2.0 ** -18 * a.abs() + E * r[rows].double().abs())


def test_one_gradient():
    n = 2 ** 31 + 12345
    t = torch.full((n,), 2.0 ** -10, device="cuda", dtype=torch.bfloat16)
    t[-1] = 2.0
    want = ((n - 1) * 2.0 ** -20 + 4.0) ** 0.5
    norm = bg.clip_grads_b200([t], want / 2)
    assert abs(float(norm) - want) <= 2.0 ** -21 * want
    # (a half but for the 1e-6 beside the norm: rounded to the power of two below)
    assert bool((t[:-1] == 2.0 ** -11).all()) and float(t[-1]) == 1.0
