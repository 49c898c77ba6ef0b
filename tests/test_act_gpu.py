"""Products with bias, activation and residual, on every kernel, against 64 bits.

Tolerances.  u is the unit roundoff of the operands' type (2^-8 bf16, 2^-11 fp16), e =
2^-24 that of fp32.  z = a b + bias is off by ez = e (K + 2) S, S the sum of its terms'
magnitudes.  The activations' slopes, and those of their slopes, are at most 1.13, and both
are evaluated within 2^-18 of their value (2^-20 besides, where that is small).
  y = act(z) + r:  u |y| + 1.13 ez + 2^-18 |act(z)| + e |r|
  dz = dy act'(z): |dy| (1.13 ez + 2^-18 |act'| + 2^-20) and, rounded for the products, u |dz|
  dA, dB, dbias: u of the result, the sum of what the terms of dz are off by (dbias: before
  their rounding), and e R S for a sum of R terms.
relu's slope jumps at 0: where |z| <= ez it may be either."""
import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi
from test_gated_gpu import BEND, DT, E, KERNELS, curve, within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean():
    capi.device_status(True)
    yield
    capi.ffn_set_kernel(0)
    assert capi.device_status(True) == 0


def check(m, n, k, dtype="bf16", act="gelu", bias=True, residual=True, seed=0,
          train=("x", "w", "b", "r"), mangle=lambda t: t):
    dt, u, tiny = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*s, scale=1.0):
        return mangle((torch.randn(*s, generator=g, device="cuda") * scale).to(dt))

    ops = {"x": randn(m, k), "w": randn(n, k, scale=max(k, 1) ** -0.5),
           "b": randn(n) if bias else None, "r": randn(m, n) if residual else None}
    dy = randn(m, n)
    leaves = [v for v in train if ops[v] is not None]
    for v in leaves:
        ops[v].requires_grad_(True)
    y = bg.matmul_b200_act(ops["x"], ops["w"].t(), ops["b"], ops["r"], activation=act)
    assert y.shape == (m, n) and y.dtype == dt and y.is_contiguous()
    grads = dict(zip(leaves, torch.autograd.grad(y, [ops[v] for v in leaves], dy))) if leaves else {}
    x, w = ops["x"].detach().double(), ops["w"].detach().double()
    b = ops["b"].detach().double() if bias else torch.zeros(n, device="cuda", dtype=torch.float64)
    r = ops["r"].detach().double() if residual else torch.zeros(m, n, device="cuda",
                                                                 dtype=torch.float64)
    z = x @ w.T + b
    ez = E * (k + 2) * (x.abs() @ w.abs().T + b.abs())
    a, slope = curve(act, z)
    within(y, a + r, u * (a + r).abs() + BEND * ez + 2.0 ** -18 * a.abs() + E * r.abs() + tiny, "y")
    d = dy.double()
    dz = d * slope
    loose = d.abs() * (BEND * ez + 2.0 ** -18 * slope.abs() + 2.0 ** -20)
    if act == "relu":
        loose = loose + d.abs() * (z.abs() <= ez)
    if act == "none":
        loose, rounded = torch.zeros_like(d), torch.zeros_like(d)
    else:
        rounded = loose + u * (dz.abs() + loose) + tiny
    if "x" in grads:
        want = dz @ w
        within(grads["x"], want, u * want.abs() + rounded @ w.abs() +
               E * (n + 1) * (dz.abs() @ w.abs()) + tiny, "dx")
    if "w" in grads:
        want = dz.T @ x
        within(grads["w"], want, u * want.abs() + rounded.T @ x.abs() +
               E * (m + 1) * (dz.abs().T @ x.abs()) + tiny, "dw")
    if "b" in grads:
        want = dz.sum(0)
        within(grads["b"], want, u * want.abs() + loose.sum(0) + E * (m + 1) * dz.abs().sum(0) + tiny,
               "db")
    if "r" in grads:
        assert torch.equal(grads["r"], dy)
    for v in leaves:
        assert grads[v].shape == ops[v].shape and grads[v].dtype == dt
    return y, grads


@pytest.mark.parametrize("kernel", list(KERNELS))
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("m,n,k", [(1, 128, 64), (1, 200, 520), (15, 136, 72), (33, 96, 256),
                                   (64, 1000, 128), (65, 264, 88), (257, 136, 320),
                                   (300, 520, 1032), (1023, 72, 200)])
def test_sizes(m, n, k, dtype, kernel):
    capi.ffn_set_kernel(KERNELS[kernel])
    check(m, n, k, dtype)


@pytest.mark.parametrize("kernel", ["stream", "pair", "cluster"])
@pytest.mark.parametrize("act", capi.ACTIVATIONS)
def test_activations(act, kernel):
    capi.ffn_set_kernel(KERNELS[kernel])
    for dtype in DT:
        for bias in (False, True):
            for residual in (False, True):
                check(70, 136, 264, dtype, act, bias, residual)


@pytest.mark.parametrize("kernel", ["stream", "pair", "cluster"])
@pytest.mark.parametrize("n,k", [(1, 1), (1, 64), (7, 9), (65, 33), (127, 515), (257, 100), (130, 6)])
def test_odd_sizes(n, k, kernel):
    capi.ffn_set_kernel(KERNELS[kernel])
    check(37, n, k)
    check(37, n, k, "fp16", "none", seed=2)


@pytest.mark.parametrize("act", ["none", "gelu", "sigmoid"])
@pytest.mark.parametrize("m,n,k", [(0, 64, 64), (5, 0, 64), (5, 64, 0), (0, 0, 0), (300, 33, 0)])
def test_empty(m, n, k, act):
    check(m, n, k, act=act)


@pytest.mark.parametrize("train", [("x",), ("w",), ("b",), ("r",), ("b", "r"), ("x", "b"), ()])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_some_gradients(act, train):
    check(100, 136, 72, act=act, train=train)


# a sum over many rows: blocks of them, added in order
@pytest.mark.parametrize("m,n", [(20000, 8), (5000, 300)])
def test_bias_of_many_rows(m, n):
    check(m, n, 16, train=("b",))
    first = check(m, n, 16, train=("b",))[1]["b"]
    assert torch.equal(first, check(m, n, 16, train=("b",))[1]["b"])


# few tiles with long contractions, divided over a cluster, in each of the three products
@pytest.mark.parametrize("m,n,k", [(70, 136, 5000), (300, 520, 2056), (257, 3208, 1608),
                                   (2000, 264, 136), (4100, 136, 72), (1, 256, 8192)])
@pytest.mark.parametrize("kernel", [2, 3])
def test_divided(m, n, k, kernel):
    capi.ffn_set_kernel(kernel)
    y, g = check(m, n, k)
    y2, g2 = check(m, n, k)
    assert torch.equal(y, y2) and all(torch.equal(g[v], g2[v]) for v in g)
