"""Routings that were changed after route_b200: slots taken out (a limit on an
expert's rows), rows out of range, rows past the last owned one.

A sorted row that no slot names is zero in what dispatch_b200 makes and in
combine_b200's gradient; every named row is served.  Rows move exactly, so
results are compared bit for bit; out-sums and dots against 64 bits."""
import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean():
    yield
    assert capi.device_status(True) == 0


def poison(*shape, dtype):
    """The allocator hands the next tensor of this size memory full of NaN."""
    torch.full(shape, float("nan"), dtype=dtype, device="cuda")


def changed(t, e, k, change, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn(t, e, generator=g, device="cuda")
    logits[::5] = -float("inf")       # tokens without an expert
    r = bg.route_b200(logits, k)
    rows = r.rows.clone()
    if change == "dropped":
        rows[torch.rand(t, k, generator=g, device="cuda") < 0.3] = -1
    elif change == "outside":
        rows[::3] = t * k + rows[::3].abs()
        rows[1::7] = -5
    elif change == "all":
        rows[:] = -1
    elif change == "moved":           # past the owned rows too
        to = torch.randperm(t * k, generator=g, device="cuda")[:t * k].int()
        rows = torch.where(rows >= 0, to[rows.clamp(min=0).long()], rows)
    return r._replace(rows=rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("change", ["none", "dropped", "outside", "all", "moved"])
@pytest.mark.parametrize("t,e,k,width", [(1, 4, 2, 64), (17, 8, 2, 72), (33, 8, 3, 30),
                                         (513, 64, 4, 256), (700, 16, 3, 2056), (1500, 40, 32, 24)])
def test_rows_nobody_names_are_zero(t, e, k, width, change, dtype):
    r = changed(t, e, k, change)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(t, width, generator=g, device="cuda").to(dtype).requires_grad_()
    y = torch.randn(t * k, width, generator=g, device="cuda").to(dtype).requires_grad_()
    w = torch.rand(t, k, generator=g, device="cuda").requires_grad_()
    dout = torch.randn(t, width, generator=g, device="cuda").to(dtype)
    ok = (r.rows >= 0) & (r.rows < t * k)
    token, slot = ok.nonzero(as_tuple=True)
    row = r.rows[ok].long()

    poison(t * k, width, dtype=dtype)
    xs = bg.dispatch_b200(x, r)
    want = torch.zeros_like(xs)
    want[row] = x.detach()[token]
    assert torch.equal(xs, want)

    out = bg.combine_b200(y, r, w)
    poison(t * k, width, dtype=dtype)
    dy, dw = torch.autograd.grad(out, (y, w), dout)
    want = torch.zeros_like(dy)
    want[row] = (w.detach()[token, slot][:, None] * dout.float()[token]).to(dtype)
    assert torch.equal(dy, want)
    dots = torch.zeros(t, k, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(dots)
    dots[ok] = (dout.double()[token] * y.detach().double()[row]).sum(1)
    size[ok] = (dout.double()[token] * y.detach().double()[row]).abs().sum(1)
    assert bool(((dw.double() - dots).abs() <= 2.0 ** -24 * (width + 8) * size).all())
    assert not dw[~ok].any()
