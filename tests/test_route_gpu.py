"""Routing, dispatch and combine against the definition, token by token, in 64 bits.

Whole numbers are exact.  Weights: exp, a sum of E terms and a quotient in
fp32, each within 2^-22 relative, and the rounding of l - max, which moves exp
by 2^-24 |l - max|; so (E + 8 + |l - max|) 2^-22 w.  Rows: fp32 sums of at
most n products, rounded once to u = 2^-8 (bf16) or 2^-11 (fp16): u |y| + (n +
2) 2^-24 sum |terms| (+ half the smallest fp16 step)."""
import numpy as np
import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi

pytestmark = pytest.mark.gpu

DT = {"bf16": (torch.bfloat16, 2.0 ** -8, 0.0), "fp16": (torch.float16, 2.0 ** -11, 2.0 ** -25)}
INF = float("inf")


@pytest.fixture(autouse=True)
def _clean():
    capi.device_status(True)
    yield
    assert capi.device_status(True) == 0


def reference(logits, k, normalize):
    """weights, experts, rows, tokens, offsets and the shares p, in numpy."""
    x = logits.double().cpu().numpy()
    t, e = x.shape
    w, ex = np.zeros((t, k)), np.full((t, k), -1)
    p = np.zeros((t, e))
    for i in range(t):
        order = sorted((j for j in range(e) if x[i, j] > -INF), key=lambda j: (-x[i, j], j))[:k]
        if not order:
            continue
        v = np.exp(x[i] - x[i, order[0]])
        if normalize:
            v = np.where(np.isin(np.arange(e), order), v, 0)
        p[i] = v / v.sum()
        w[i, :len(order)], ex[i, :len(order)] = p[i, order], order
    rows, tokens, offsets = np.full((t, k), -1), np.full(t * k, -1), [0]
    at = 0
    for j in range(e):
        for i, s in zip(*np.nonzero(ex == j)):      # by token, then slot
            rows[i, s], tokens[at] = at, i
            at += 1
        offsets.append(at)
    return w, ex, rows, tokens, np.array(offsets), p


def check(logits, k, normalize):
    r = bg.route_b200(logits, k, normalize=normalize)
    w, ex, rows, tokens, offsets, p = reference(logits, k, normalize)
    assert np.array_equal(r.experts.cpu().numpy(), ex)
    assert np.array_equal(r.rows.cpu().numpy(), rows)
    assert np.array_equal(r.tokens.cpu().numpy(), tokens)
    assert np.array_equal(r.offsets.cpu().numpy(), offsets)
    x = logits.double().cpu().numpy()
    top = np.where(np.isfinite(x), x, -INF).max(1, keepdims=True)
    span = np.where(ex >= 0, top - np.take_along_axis(x, np.maximum(ex, 0), 1), 0)
    off = np.abs(r.weights.double().cpu().numpy() - w)
    assert (off <= (logits.shape[1] + 8 + span) * 2.0 ** -22 * w + 1e-44).all(), off.max()
    return r


def make(t, e, seed, closed=0.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(t, e, generator=g, device="cuda") * 2
    if closed:
        x[torch.rand(t, e, generator=g, device="cuda") < closed] = -INF
        x[::5] = -INF
    return x.to(dtype)


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 8, 2), (7, 4, 4), (33, 60, 6), (256, 64, 4),
                                   (257, 64, 4), (300, 129, 8), (600, 257, 3), (40, 1024, 32),
                                   (1500, 33, 2)])
def test_sizes(t, e, k, normalize):
    check(make(t, e, t + e), k, normalize)
    check(make(t, e, t + e, closed=0.6), k, normalize)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_types_and_ties(dtype):
    x = make(400, 32, 0, dtype=dtype)
    x = (x * 2).round() / 2           # many equal logits: the lower index first
    check(x, 4, True)
    check(x, 4, False)
    check(torch.zeros(290, 40, device="cuda", dtype=dtype), 7, True)
    signed = torch.zeros(3, 8, device="cuda", dtype=dtype)
    signed[:, ::2] = -0.0             # -0 and +0 are equal
    check(signed, 3, True)


def test_masks_and_odd_values():
    low = torch.finfo(torch.float32).min
    x = make(6, 8, 1)
    x[0] = -INF
    x[1] = low                        # open, however low: a uniform row
    x[2, 1:] = low                    # one open in effect: the others weigh 0
    x[3, :7] = -INF                   # one open: an empty slot
    check(x, 3, True)
    check(x, 3, False)
    nan = float("nan")
    y = torch.tensor([[0.0, nan, 3.0, nan], [INF, 1.0, INF, 2.0]], device="cuda")
    r = bg.route_b200(y, 3)
    assert r.experts.tolist() == [[1, 3, 2], [0, 2, 3]]
    assert bool(r.weights[0].isnan().all()) and bool(r.weights[1].isnan().all())


def test_strided_logits_and_empty():
    wide = make(300, 64, 3)
    check(wide[:, 5:45], 4, True)
    assert torch.equal(bg.route_b200(wide.t().contiguous().t(), 4).rows,
                       bg.route_b200(wide, 4).rows)
    r = bg.route_b200(wide[:0], 4)
    assert r.rows.shape == (0, 4) and r.tokens.shape == (0,) and not r.offsets.any()
    x = torch.zeros(0, 16, dtype=torch.bfloat16, device="cuda")
    assert bg.dispatch_b200(x, r).shape == (0, 16) and bg.combine_b200(x, r).shape == (0, 16)


def test_many_tokens_order():
    # (by sorting: the token-by-token reference is slow at this size)
    x = make(20001, 48, 4)
    r = bg.route_b200(x, 3)
    flat = r.experts.flatten().long()
    order = torch.argsort(flat, stable=True)
    assert torch.equal(r.tokens.long(), order // 3)
    want = torch.empty_like(order)
    want[order] = torch.arange(order.numel(), device="cuda")
    assert torch.equal(r.rows.flatten().long(), want)
    assert torch.equal(r.offsets[1:].long(), torch.bincount(flat, minlength=48).cumsum(0))


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("e,k", [(8, 2), (70, 5), (300, 32)])
def test_route_gradient(e, k, normalize):
    x = make(37, e, e, closed=0.3).requires_grad_(True)
    r = bg.route_b200(x, k, normalize=normalize)
    g = torch.randn(37, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    dx, = torch.autograd.grad(r.weights, x, g)
    w, ex, _, _, _, p = reference(x.detach(), k, normalize)
    gd = np.where(ex >= 0, g.double().cpu().numpy(), 0)
    hit = np.zeros((37, e))
    for j in range(k):
        ok = ex[:, j] >= 0
        hit[ok, ex[ok, j]] = gd[ok, j]
    inner = (w * gd).sum(1, keepdims=True)
    want = p * (hit - inner)
    # relative 2^-22 (2 E + 16) of p (|hit| + sum |w g|), by the same count as the weights
    size = p * (np.abs(hit) + (w * np.abs(gd)).sum(1, keepdims=True))
    off = np.abs(dx.double().cpu().numpy() - want)
    assert (off <= (2 * e + 32) * 2.0 ** -22 * size + 1e-44).all()
    # differences of the definition itself
    h = 1e-5
    xd = x.detach().double().cpu().numpy()
    for i, j in ((1, 0), (2, e - 1), (3, e // 2)):
        if not np.isfinite(xd[i, j]):
            continue
        def f(v):
            y = torch.from_numpy(xd[i:i + 1].copy())
            y[0, j] += v
            ww, ee = reference(y, k, normalize)[:2]
            assert np.array_equal(ee, ex[i:i + 1])
            return float((ww * gd[i:i + 1]).sum())
        slope = (f(h) - f(-h)) / (2 * h)
        assert abs(slope - want[i, j]) <= 1e-6 * max(1.0, abs(slope))


def rows_close(got, want, size, n, u, tiny):
    off = (got.double() - want).abs() - (1.0001 * u * want.abs() + (n + 2) * 2.0 ** -24 * size + tiny)
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("t,e,k,width", [(1, 4, 1, 8), (5, 8, 2, 4096), (64, 16, 8, 264),
                                         (300, 64, 4, 1001), (9, 8, 3, 1), (70, 40, 32, 2048)])
def test_rows_there_and_back(t, e, k, width, dtype):
    dt, u, tiny = DT[dtype]
    logits = make(t, e, width, closed=0.4).requires_grad_(True)
    g = torch.Generator(device="cuda").manual_seed(t)

    def randn(*s):
        return torch.randn(*s, generator=g, device="cuda").to(dt)

    x, y = randn(t, width).requires_grad_(True), randn(t * k, width).requires_grad_(True)
    dxs, dout = randn(t * k, width), randn(t, width)
    r = bg.route_b200(logits, k)
    xs = bg.dispatch_b200(x, r)
    total = int(r.offsets[-1])
    assert torch.equal(xs[:total], x[r.tokens[:total].long()]) and not xs[total:].any()
    # rows of no expert may hold anything
    yb = y.detach().clone()
    yb[total:] = float("nan")
    yb.requires_grad_(True)
    w = r.weights.detach().requires_grad_(True)
    out = bg.combine_b200(yb, r, w)
    mine = r.rows >= 0
    picked = torch.where(mine[..., None], y.detach().double()[r.rows.clamp(min=0).long()], 0)
    terms = w.detach().double()[..., None] * picked
    rows_close(out, terms.sum(1), terms.abs().sum(1), k, u, tiny)
    dx, = torch.autograd.grad(xs, x, dxs)
    back = torch.where(mine[..., None], dxs.double()[r.rows.clamp(min=0).long()], 0)
    rows_close(dx, back.sum(1), back.abs().sum(1), k, u, tiny)
    dy, dw = torch.autograd.grad(out, (yb, w), dout)
    want = torch.zeros(t * k, width, dtype=torch.float64, device="cuda")
    wide = w.detach().double()[..., None] * dout.double()[:, None]
    want[r.rows[mine].long()] = wide[mine]
    rows_close(dy, want, want.abs(), 1, u, tiny)
    dots = dout.double()[:, None] * picked
    off = (dw.double() - dots.sum(2)).abs()
    assert bool((off <= (width + 2) * 2.0 ** -24 * dots.abs().sum(2) + 1e-44).all())
    # the whole chain reaches the logits
    bg.combine_b200(yb.detach(), r).backward(dout)
    assert logits.grad is not None and bool(logits.grad.isfinite().all())


def test_strided_and_unaligned_rows():
    r = bg.route_b200(make(50, 8, 1), 2)
    x = torch.randn(50, 256, device="cuda").bfloat16()
    y = torch.randn(100, 256, device="cuda").bfloat16()
    xs, out = bg.dispatch_b200(x, r), bg.combine_b200(y, r)
    for pad, at in ((16, 8), (3, 1)):
        for src, fn, want in ((x, bg.dispatch_b200, xs), (y, bg.combine_b200, out)):
            wide = torch.zeros(src.shape[0], 256 + pad, dtype=torch.bfloat16, device="cuda")
            wide[:, at:at + 256] = src
            assert torch.equal(fn(wide[:, at:at + 256], r), want)
            assert torch.equal(fn(src.t().contiguous().t(), r), want)


def test_rows_out_of_range_are_skipped():
    r = bg.route_b200(make(4, 8, 1), 2)
    rows = r.rows.clone()
    rows[0, 0], rows[1, 1] = 8, -7
    bad = r._replace(rows=rows)
    y = torch.ones(8, 16, dtype=torch.bfloat16, device="cuda")
    ones = torch.ones(4, 2, device="cuda")
    assert bg.combine_b200(y, bad, ones)[:, 0].tolist() == [1, 1, 2, 2]
    assert bg.dispatch_b200(y[:4], bad).shape == (8, 16)


def test_refusals():
    x = make(4, 8, 0)
    for bad, match in ((x.double(), "float32"), (x[0], "tokens, experts"),
                       (torch.zeros(2, 1025, device="cuda"), "1024 experts")):
        with pytest.raises(RuntimeError, match=match):
            bg.route_b200(bad, 1)
    for k in (0, 9, -1):
        with pytest.raises(RuntimeError, match="top_k"):
            bg.route_b200(x, k)
    with pytest.raises(RuntimeError, match="top_k"):
        bg.route_b200(torch.zeros(2, 64, device="cuda"), 33)
    r = bg.route_b200(x, 2)
    rows = torch.zeros(4, 16, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="the routing 4"):
        bg.dispatch_b200(rows[:3], r)
    with pytest.raises(RuntimeError, match="the routing 8"):
        bg.combine_b200(rows, r)
    with pytest.raises(RuntimeError, match="bfloat16 or float16"):
        bg.dispatch_b200(rows.float(), r)
    with pytest.raises(RuntimeError, match="weights must be float32"):
        bg.combine_b200(torch.cat((rows, rows)), r, r.weights.bfloat16())
    with pytest.raises(RuntimeError, match="must come from route_b200"):
        bg.dispatch_b200(rows, r._replace(rows=r.rows.long()))


def test_graph_capture():
    x, y = make(700, 16, 0), torch.randn(1400, 64, device="cuda").bfloat16()

    def step():
        r = bg.route_b200(x, 2)
        return (*r, bg.combine_b200(y, r))

    want = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
