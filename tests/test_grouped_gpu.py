"""Products grouped by expert, forward and both gradients, on every kernel,
against expert-by-expert products in 64 bits.

Tolerance: an output is one fp32 sum of R products rounded once.  With u the
unit roundoff of the output type (2^-8 bf16, 2^-11 fp16: half a spacing), the
error is at most u |y| from the rounding plus the fp32 summation error, which
for any order of adding is within 2^-24 * R * sum |a b|; that worst case is
used as it stands."""
import numpy as np
import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi

pytestmark = pytest.mark.gpu

DT = {"bf16": (torch.bfloat16, 2.0 ** -8), "fp16": (torch.float16, 2.0 ** -11)}
KERNELS = {"chosen": 0, "stream": 1, "pair": 2}


@pytest.fixture(autouse=True)
def _clean():
    capi.device_status(True)
    yield
    capi.grouped_set_kernel(0)
    assert capi.device_status(True) == 0


def close(got, want, size, terms, u, tiny):
    """|got - want| <= u |want| + 2^-24 terms size (size = the sum of |a b|)."""
    bound = 1.0001 * u * want.abs() + 2.0 ** -24 * terms * size + tiny
    off = (got.double() - want).abs() - bound
    assert bool((off <= 0).all()), float(off.max())


def spans(offsets):
    return [(e, offsets[e], offsets[e + 1]) for e in range(len(offsets) - 1)]


def operands(offsets, rows, n, k, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, k, generator=g, device="cuda").to(dt)
    w = (torch.randn(len(offsets) - 1, n, k, generator=g, device="cuda") * k ** -0.5).to(dt)
    dy = torch.randn(rows, n, generator=g, device="cuda").to(dt)
    return x, w, dy, torch.tensor(offsets, dtype=torch.int32, device="cuda")


def check_all(offsets, rows, n, k, dtype="bf16", seed=0, mangle=lambda t: t):
    dt, u = DT[dtype]
    tiny = 2.0 ** -25 if dtype == "fp16" else 0.0   # half the smallest fp16 step
    x, w, dy, off = operands(offsets, rows, n, k, dt, seed)
    xg, wg = mangle(x).requires_grad_(True), mangle(w).requires_grad_(True)
    y = bg.matmul_b200_grouped(xg, wg.transpose(1, 2), off)
    assert y.shape == (rows, n) and y.dtype == dt and y.is_contiguous()
    dx, dw = torch.autograd.grad(y, (xg, wg), mangle(dy))
    owned = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for e, a, b in spans(offsets):
        owned[a:b] = True
        xe, we, de = x[a:b].double(), w[e].double(), dy[a:b].double()
        close(y[a:b], xe @ we.T, xe.abs() @ we.abs().T, k, u, tiny)
        close(dx[a:b], de @ we, de.abs() @ we.abs(), n, u, tiny)
        close(dw[e], de.T @ xe, de.abs().T @ xe.abs(), max(b - a, 1), u, tiny)
    assert not y[~owned].any() and not dx[~owned].any()


# rows per expert: none, one, around the 16-, 32-, 64- and 256-row edges
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
    offsets, rows = LAYOUTS[layout]
    capi.grouped_set_kernel(KERNELS[kernel])
    check_all(offsets, rows, 264, 200, dtype)


@pytest.mark.parametrize("kernel", list(KERNELS))
@pytest.mark.parametrize("n,k", [(1, 1), (8, 8), (7, 129), (130, 63), (256, 64), (257, 320),
                                 (1000, 17), (24, 1000), (640, 2048)])
def test_odd_sizes(n, k, kernel):
    capi.grouped_set_kernel(KERNELS[kernel])
    check_all([0, 5, 5, 70, 81], 83, n, k, "bf16", seed=n + k)


def test_many_experts():
    r = np.random.default_rng(0)
    counts = r.integers(0, 5, 1024)
    counts[r.integers(0, 1024, 700)] = 0
    offsets = np.concatenate([[0], np.cumsum(counts)]).tolist()
    check_all(offsets, offsets[-1], 72, 136)
    capi.grouped_set_kernel(2)
    check_all(offsets, offsets[-1], 72, 136)


def test_long_group_and_wide_output():
    check_all([0, 40, 2600, 2600, 5001], 5001, 1288, 776, "bf16")


def test_strided_operands():
    # column slices of wider buffers (aligned rows), and unaligned ones
    def aligned(t):
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 24, dtype=t.dtype, device=t.device)
        wide[..., 8:8 + t.shape[-1]] = t
        return wide[..., 8:8 + t.shape[-1]].detach()

    def unaligned(t):
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
        wide[..., 1:1 + t.shape[-1]] = t
        return wide[..., 1:1 + t.shape[-1]].detach()

    def transposed(t):
        return t.transpose(-1, -2).contiguous().transpose(-1, -2).detach()

    for mangle in (aligned, unaligned, transposed):
        check_all([0, 30, 94, 101], 101, 128, 192, mangle=mangle)


def test_expanded_gradient_and_int64_offsets():
    x, w, _, off = operands([0, 9, 20], 20, 64, 64, torch.bfloat16)
    w.requires_grad_(True)
    y = bg.matmul_b200_grouped(x, w.transpose(1, 2), off.long())
    y.sum().backward()      # the incoming gradient has stride 0
    for e, a, b in spans([0, 9, 20]):
        want = x[a:b].double().sum(0).expand(64, 64)
        close(w.grad[e], want, x[a:b].double().abs().sum(0).expand(64, 64), 20, 2.0 ** -8, 0.0)


@pytest.mark.parametrize("kernel", ["stream", "pair"])
def test_other_rows_stay_out(kernel):
    # inf and NaN in rows of other experts and of none, and in unused experts
    offsets, rows, n, k = [2, 37, 37, 90, 113], 120, 136, 200
    x, w, dy, off = operands(offsets, rows, n, k, torch.bfloat16)
    capi.grouped_set_kernel(KERNELS[kernel])

    def run(x, w, dy):
        xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = bg.matmul_b200_grouped(xg, wg.transpose(1, 2), off)
        return (y, *torch.autograd.grad(y, (xg, wg), dy))

    y0, dx0, dw0 = run(x, w, dy)
    bad = float("inf")
    x1, w1, dy1 = x.clone(), w.clone(), dy.clone()
    for t in (x1, dy1):
        t[:2], t[113:], t[37:90] = bad, float("nan"), bad
    w1[1], w1[2] = float("nan"), bad
    y1, dx1, dw1 = run(x1, w1, dy1)
    for e, a, b in [(0, 2, 37), (3, 90, 113)]:
        assert torch.equal(y0[a:b], y1[a:b]) and torch.equal(dx0[a:b], dx1[a:b])
        assert torch.equal(dw0[e], dw1[e])
    assert not dw1[1].any() and not y1[:2].any() and not y1[113:].any()
    assert not dx1[:2].any() and not dx1[113:].any()
    assert bool((y1[37:90] == bad).all())     # sums of inf x inf: as the product says


@pytest.mark.parametrize("kernel", ["stream", "pair"])
def test_repeatable_bits(kernel):
    x, w, dy, off = operands([0, 3, 50, 51, 120], 120, 1024, 4096, torch.bfloat16)
    capi.grouped_set_kernel(KERNELS[kernel])
    first = bg.matmul_b200_grouped(x, w.transpose(1, 2), off)
    for _ in range(20):
        assert torch.equal(first, bg.matmul_b200_grouped(x, w.transpose(1, 2), off))


def test_gradient_against_differences():
    # f = <y, c>: a step along a direction, in steps that bf16 holds exactly
    offsets = [0, 7, 7, 40]
    x, w, c, off = operands(offsets, 40, 64, 64, torch.bfloat16)
    x, w = (x * 4).round() / 4, (w * 4).round() / 4
    c = (c * 2).round() / 2
    c = c.to(torch.bfloat16)
    xg, wg = x.requires_grad_(True), w.requires_grad_(True)
    y = bg.matmul_b200_grouped(xg, wg.transpose(1, 2), off)
    dx, dw = torch.autograd.grad(y, (xg, wg), c)

    def f(x, w):
        y = torch.zeros(40, 64, dtype=torch.float64, device="cuda")
        for e, a, b in spans(offsets):
            y[a:b] = x[a:b].double() @ w[e].double().T
        return float((y * c.double()).sum())

    h = 0.25
    for t, d, at in ((x, dx, (3, 5)), (x, dx, (39, 63)), (w, dw, (0, 9, 1)), (w, dw, (2, 63, 0)),
                     (w, dw, (1, 4, 4))):
        up, down = t.detach().clone(), t.detach().clone()
        up[at] += h
        down[at] -= h
        a = (up, w) if t is x else (x, up)
        b = (down, w) if t is x else (x, down)
        slope = (f(*(v.detach() for v in a)) - f(*(v.detach() for v in b))) / (2 * h)
        assert abs(float(d[at]) - slope) <= 2.0 ** -8 * abs(slope) + 1e-9


def test_empty_extents():
    off = torch.tensor([0, 4, 6], dtype=torch.int32, device="cuda")

    def zeros(*s):
        return torch.zeros(*s, dtype=torch.bfloat16, device="cuda")

    y = bg.matmul_b200_grouped(zeros(6, 0), zeros(2, 0, 5), off)
    assert y.shape == (6, 5) and not y.any()
    assert bg.matmul_b200_grouped(zeros(6, 8), zeros(2, 8, 0), off).shape == (6, 0)
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    x, w = zeros(0, 16).requires_grad_(True), (zeros(2, 8, 16) + 1).requires_grad_(True)
    y = bg.matmul_b200_grouped(x, w.transpose(1, 2), none)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == (0, 8) and dx.shape == (0, 16) and dw.shape == (2, 8, 16) and not dw.any()
    no_expert = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = bg.matmul_b200_grouped(zeros(4, 16), zeros(0, 16, 8), no_expert)
    assert y.shape == (4, 8) and not y.any()


def test_bad_offsets_are_clamped_and_reported():
    x, w, _, _ = operands([0, 9, 20], 20, 64, 64, torch.bfloat16)
    for bad in ([0, 12, 30], [0, 15, 10], [-4, 3, 20]):
        for kernel in (1, 2):
            capi.grouped_set_kernel(kernel)
            off = torch.tensor(bad, dtype=torch.int32, device="cuda")
            y = bg.matmul_b200_grouped(x, w.transpose(1, 2), off)
            assert capi.device_status(True) == 0x100A
            a = min(max(bad[0], 0), 20)
            b = max(min(bad[1], 20), a)
            size = x[a:b].double().abs() @ w[0].double().abs().T
            close(y[a:b], x[a:b].double() @ w[0].double().T, size, 64, 2.0 ** -8, 0.0)


def test_other_stream_and_graph_capture():
    x, w, _, off = operands([0, 3, 60, 61, 100], 100, 512, 2048, torch.bfloat16)
    want = bg.matmul_b200_grouped(x, w.transpose(1, 2), off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = bg.matmul_b200_grouped(x, w.transpose(1, 2), off)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    static = x.clone()
    with torch.cuda.graph(graph):
        y = bg.matmul_b200_grouped(static, w.transpose(1, 2), off)
    for scale in (1.0, 2.0):
        static.copy_(x * scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, bg.matmul_b200_grouped(static, w.transpose(1, 2), off))


def test_rows_anywhere():
    # odd strides and starts in every operand that is read
    def odd(t, pad):
        wide = torch.full((*t.shape[:-1], t.shape[-1] + pad), float("nan"), dtype=t.dtype,
                          device=t.device)
        wide[..., pad // 2:pad // 2 + t.shape[-1]] = t
        return wide[..., pad // 2:pad // 2 + t.shape[-1]].detach()

    for n, k in ((33, 75), (64, 129), (131, 64), (9, 7)):
        for pad in (1, 2, 5):
            check_all([0, 30, 94, 101], 101, n, k, seed=pad, mangle=lambda t: odd(t, pad))


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 8), (17, 9), (64, 1033), (300, 250)])
def test_align_rows(rows, cols):
    from blackwell_gemm_b200 import capi as c
    ld = (cols + 7) // 8 * 8
    for stride in (cols, cols + 1, cols + 6):
        for start in (0, 1, 2, 3, 7):
            flat = torch.randn(2 * rows * stride + 8, device="cuda").bfloat16()
            src = torch.as_strided(flat, (2, rows, cols), (rows * stride, stride, 1), start)
            dst = torch.full((2, rows, ld), 9.0, device="cuda").bfloat16()
            st = c.lib().b200_align_rows(src.data_ptr(), rows * stride, stride, dst.data_ptr(), 2,
                                         rows, cols, ld, torch.cuda.current_stream().cuda_stream)
            assert st == c.OK
            assert torch.equal(dst[..., :cols], src) and not dst[..., cols:].any()
