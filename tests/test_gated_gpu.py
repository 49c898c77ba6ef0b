"""Gated products, dense and by expert, on every kernel, against products in 64 bits.

Tolerances.  u is the unit roundoff of the operands' type (2^-8 bf16, 2^-11 fp16),
e = 2^-24 that of fp32.  A product of R terms is off by at most e R S, S the sum of the
terms' magnitudes, in any order of adding.

h = act(g) u: with dg = e K Sg and du = e K Su the products' errors, and act having a
slope of at most 1.13 and evaluated within 2^-18 of its value, |dh| <= u |h| +
(1.13 dg + 2^-18 |act|) |u| + |act| du + 1.13 dg du.

The gradients round dg, du once (u of their value) and sum with 16-bit operands:
|error| <= u |result| + (u + 2^-17) S + the fp32 sums' e R S, S the sum of the magnitudes
of the result's terms, to which the error of the products g and u adds its share: slopes and
act bend by at most 1.13, so a term dh u act'(g) moves by at most |dh| (du 1.13 + |u| 1.13
dg), and |dh act(g)| by |dh| 1.13 dg.  relu's slope jumps at 0: where |g| <= dg it may be
either."""
import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi

pytestmark = pytest.mark.gpu

DT = {"bf16": (torch.bfloat16, 2.0 ** -8, 0.0), "fp16": (torch.float16, 2.0 ** -11, 2.0 ** -25)}
KERNELS = {"chosen": 0, "stream": 1, "pair": 2, "cluster": 3}
E = 2.0 ** -24
BEND = 1.13  # the largest slope of the activations, and of their slopes


@pytest.fixture(autouse=True)
def _clean():
    capi.device_status(True)
    yield
    capi.ffn_set_kernel(0)
    assert capi.device_status(True) == 0


def curve(name, z):
    """act(z) and act'(z) in 64 bits.  (gelu by erfc and its tanh form by the logistic
    function: 1 + erf and 1 + tanh leave nothing of their tails even in 64 bits.)"""
    z = z.detach().clone().requires_grad_(True)
    f = {"none": lambda t: t * 1, "relu": torch.relu, "silu": torch.nn.functional.silu,
         "gelu": lambda t: t * torch.special.erfc(t * -0.5 ** 0.5) / 2, "sigmoid": torch.sigmoid,
         "gelu_tanh": lambda t: t * torch.sigmoid((8 / torch.pi) ** 0.5 * (t + 0.044715 * t ** 3))}[name]
    a = f(z)
    return a.detach(), torch.autograd.grad(a.sum(), z)[0]


def within(got, want, bound, name=""):
    off = (got.double() - want).abs() - 1.0001 * bound
    assert bool((off <= 0).all()), (name, float(off.max()))


def spans(offsets, rows):
    if offsets is None:
        return [(None, 0, rows)]
    return [(e, offsets[e], offsets[e + 1]) for e in range(len(offsets) - 1)]


def check(offsets, rows, n, k, dtype="bf16", act="silu", seed=0, train=True, mangle=lambda t: t,
          off_dtype=torch.int32):
    dt, u, tiny = DT[dtype]
    bank = () if offsets is None else (len(offsets) - 1,)
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*s, scale=1.0):
        return mangle((torch.randn(*s, generator=g, device="cuda") * scale).to(dt))

    x, wg, wu, dh = (randn(rows, k), randn(*bank, n, k, scale=max(k, 1) ** -0.5),
                     randn(*bank, n, k, scale=max(k, 1) ** -0.5), randn(rows, n))
    off = None if offsets is None else torch.tensor(offsets, dtype=off_dtype, device="cuda")
    if train:
        for t in (x, wg, wu):
            t.requires_grad_(True)
    h = bg.matmul_b200_gated(x, wg.transpose(-1, -2), wu.transpose(-1, -2), off, activation=act)
    assert h.shape == (rows, n) and h.dtype == dt and h.is_contiguous()
    grads = torch.autograd.grad(h, (x, wg, wu), dh) if train else None
    owned = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for e, a, b in spans(offsets, rows):
        owned[a:b] = True
        xe, de = x[a:b].detach().double(), dh[a:b].double()
        ge, ue = ((t if e is None else t[e]).detach().double() for t in (wg, wu))
        gs, us = xe @ ge.T, xe @ ue.T
        eg, eu = E * (k + 1) * (xe.abs() @ ge.abs().T), E * (k + 1) * (xe.abs() @ ue.abs().T)
        y, slope = curve(act, gs)
        bound = (u * (y * us).abs() + (BEND * eg + 2.0 ** -18 * y.abs()) * us.abs() + y.abs() * eu
                 + BEND * eg * eu + tiny)
        within(h[a:b], y * us, bound, "h")
        if not train:
            continue
        dg, du = de * us * slope, de * y
        # what each element of dg and du may be off by before the products
        fg = (u + 2.0 ** -17) * dg.abs() + de.abs() * BEND * (eu + us.abs() * eg + eu * eg) \
            + de.abs() * us.abs() * 2.0 ** -20 + tiny
        if act == "relu":
            fg = fg + (1 + u) * (de * us).abs() * (gs.abs() <= eg)
        fu = (u + 2.0 ** -17) * du.abs() + de.abs() * BEND * eg + de.abs() * 2.0 ** -20 * y.abs() + tiny
        want = dg @ ge + du @ ue
        size = dg.abs() @ ge.abs() + du.abs() @ ue.abs()
        within(grads[0][a:b], want,
               u * want.abs() + fg @ ge.abs() + fu @ ue.abs() + E * 2 * (n + 1) * size + tiny, "dx")
        for got, d, f in ((grads[1], dg, fg), (grads[2], du, fu)):
            want = d.T @ xe
            within(got if e is None else got[e], want,
                   u * want.abs() + f.T @ xe.abs() + E * (b - a + 1) * (d.abs().T @ xe.abs()) + tiny,
                   "dw")
    assert not h[~owned].any()
    if train:
        assert not grads[0][~owned].any()
        assert [t.shape for t in grads] == [t.shape for t in (x, wg, wu)]
    return h, grads


@pytest.mark.parametrize("kernel", list(KERNELS))
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,n,k", [(1, 64, 64), (1, 200, 520), (15, 128, 72), (33, 96, 256),
                                      (64, 1000, 128), (65, 264, 88), (257, 136, 320),
                                      (300, 520, 1032), (1023, 72, 200)])
def test_dense(rows, n, k, dtype, kernel):
    capi.ffn_set_kernel(KERNELS[kernel])
    check(None, rows, n, k, dtype)


LAYOUTS = {
    "one_row": ([0, 0, 1, 1], 1),
    "edges": ([0, 1, 16, 33, 33, 97, 160, 415, 671, 928], 928),
    "unowned": ([3, 20, 20, 300], 310),
    "all_unowned": ([5, 5, 5], 12),
    "last_only": ([0, 0, 0, 0, 77], 77),
}


@pytest.mark.parametrize("kernel", list(KERNELS))
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_layouts(layout, dtype, kernel):
    capi.ffn_set_kernel(KERNELS[kernel])
    check(*LAYOUTS[layout], 136, 200, dtype)


@pytest.mark.parametrize("kernel", ["stream", "pair", "cluster"])
@pytest.mark.parametrize("act", capi.ACTIVATIONS)
def test_activations(act, kernel):
    capi.ffn_set_kernel(KERNELS[kernel])
    for dtype in DT:
        check(None, 70, 136, 264, dtype, act)
        check([0, 40, 40, 66], 70, 136, 264, dtype, act, seed=1)


# odd widths: rows that TMA and vector stores cannot take
@pytest.mark.parametrize("kernel", ["stream", "pair", "cluster"])
@pytest.mark.parametrize("n,k", [(1, 1), (1, 64), (7, 9), (65, 33), (127, 515), (257, 100), (130, 6)])
def test_odd_sizes(n, k, kernel):
    capi.ffn_set_kernel(KERNELS[kernel])
    check(None, 37, n, k)
    check([0, 20, 37], 37, n, k, "fp16", seed=2)


@pytest.mark.parametrize("rows,n,k", [(0, 64, 64), (5, 0, 64), (5, 64, 0), (0, 0, 0)])
def test_empty(rows, n, k):
    check(None, rows, n, k)
    check([0, 0, rows], rows, n, k)


# few tiles with long contractions, divided over a cluster, in each of the three products
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,n,k", [(70, 136, 5000), (300, 520, 2056), (257, 1601, 1608),
                                      (2000, 264, 136), (4100, 136, 72), (1, 256, 8192)])
@pytest.mark.parametrize("kernel", [2, 3])
def test_divided(rows, n, k, dtype, kernel):
    capi.ffn_set_kernel(kernel)
    first = check(None, rows, n, k, dtype)
    again = check(None, rows, n, k, dtype)
    assert torch.equal(first[0], again[0])     # joined in one order
    assert all(torch.equal(a, b) for a, b in zip(first[1], again[1]))


@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_divided_layouts(layout):
    capi.ffn_set_kernel(2)
    check(*LAYOUTS[layout], 1608, 2056)


# tiles left over after whole waves: their contractions divided over all pairs
@pytest.mark.parametrize("rows,n,k", [(600, 3300, 1608), (1500, 1601, 1608), (7000, 1280, 2560)])
def test_left_over(rows, n, k):
    capi.ffn_set_kernel(2)
    first = check(None, rows, n, k)
    again = check(None, rows, n, k)
    assert torch.equal(first[0], again[0])     # joined in one order
    assert all(torch.equal(a, b) for a, b in zip(first[1], again[1]))
