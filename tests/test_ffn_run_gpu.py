"""Feed-forward operators as a program runs them: a layer's training steps, strides, padding
rows that hold anything, streams, graphs, threads, derivatives, refusals on the device."""
import threading
import time

import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi
from test_act_gpu import check as check_act
from test_gated_gpu import check as check_gated
from test_gated_gpu import curve

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean():
    capi.device_status(True)
    yield
    capi.ffn_set_kernel(0)
    assert capi.device_status(True) == 0


def randn(*s, seed=0, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*s, generator=g, device="cuda") * scale).to(dtype)


# ------------------------------------------------------------------ a layer's step
@pytest.mark.parametrize("rows", [1, 33, 700])
def test_feed_forward_block(rows):
    """y = x + down(silu(x gate) * (x up)), its gradients clipped: against 64 bits.

    Six roundings to bf16 follow one another on the longest way (h, dz of the down
    product is dy itself, dh, dg, dx, the sum with the residual's gradient, the clipped value),
    each within 2^-8 of its value; the norm of the difference is at most their sum."""
    width, hidden = 264, 520
    x = randn(rows, width).requires_grad_()
    gate, up = (randn(hidden, width, seed=i, scale=width ** -0.5).requires_grad_() for i in (1, 2))
    down = randn(width, hidden, seed=3, scale=hidden ** -0.5).requires_grad_()
    dy = randn(rows, width, seed=4)
    h = bg.matmul_b200_gated(x, gate.t(), up.t())
    y = bg.matmul_b200_act(h, down.t(), residual=x)
    leaves = (x, gate, up, down)
    grads = torch.autograd.grad(y, leaves, dy)
    xd, gd, ud, dd = (t.detach().double().requires_grad_() for t in leaves)
    yd = xd + (torch.nn.functional.silu(xd @ gd.T) * (xd @ ud.T)) @ dd.T
    want = torch.autograd.grad(yd, (xd, gd, ud, dd), dy.double())
    assert float((y.detach().double() - yd.detach()).norm() / yd.detach().norm()) <= 2 * 2.0 ** -8
    norm = bg.clip_grads_b200(list(grads), 0.5)
    total = torch.stack([w.norm() for w in want]).norm()
    assert abs(float(norm) - float(total)) <= 6 * 2.0 ** -8 * float(total)
    scale = min(1.0, 0.5 / float(total))
    for g, w in zip(grads, want):
        assert float((g.double() - w * scale).norm() / (w * scale).norm()) <= 12 * 2.0 ** -8


def test_experts_layer():
    """Routed tokens through gated experts and back, with gradients, against each expert's
    rows alone."""
    tokens, experts, width, hidden = 200, 8, 128, 192
    routing = bg.route_b200(torch.randn(tokens, experts, device="cuda",
                                        generator=torch.Generator("cuda").manual_seed(0)), 2)
    x = randn(tokens, width)
    both = randn(experts, 2 * hidden, width, seed=1, scale=width ** -0.5).requires_grad_()
    xs = bg.dispatch_b200(x, routing).requires_grad_()
    # gate and up as halves of one bank
    h = bg.matmul_b200_gated(xs, both[:, :hidden].transpose(1, 2), both[:, hidden:].transpose(1, 2),
                             routing.offsets)
    dh = randn(*h.shape, seed=2)
    dxs, dboth = torch.autograd.grad(h, (xs, both), dh)
    for e in range(experts):
        a, b = int(routing.offsets[e]), int(routing.offsets[e + 1])
        xe = xs[a:b].detach().requires_grad_()
        we = both[e].detach().requires_grad_()
        he = bg.matmul_b200_gated(xe, we[:hidden].t(), we[hidden:].t())
        gx, gw = torch.autograd.grad(he, (xe, we), dh[a:b])
        # (other tiles, another order of the same fp32 sums: a last bit of bf16)
        for got, want in ((h[a:b], he), (dxs[a:b], gx), (dboth[e], gw)):
            got, want = got.detach().double(), want.detach().double()
            assert float((got - want).norm()) <= 2.0 ** -8 * float(want.norm())


# ------------------------------------------------------------------------ operands
def odd(t, pad):
    wide = torch.full((*t.shape[:-1], t.shape[-1] + pad), float("nan"), dtype=t.dtype,
                      device=t.device)
    wide[..., pad // 2:pad // 2 + t.shape[-1]] = t
    return wide[..., pad // 2:pad // 2 + t.shape[-1]].detach()


@pytest.mark.parametrize("pad", [1, 2, 5, 8])
def test_rows_anywhere(pad):
    for n, k in ((33, 75), (64, 129), (131, 64)):
        check_gated(None, 101, n, k, seed=pad, mangle=lambda t: odd(t, pad))
        check_gated([0, 30, 94, 101], 101, n, k, seed=pad, mangle=lambda t: odd(t, pad))
        check_act(101, n, k, seed=pad, mangle=lambda t: odd(t, pad))


def turned(t):
    """The same values, rows and columns exchanged in memory."""
    return t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else t


def test_turned_operands():
    check_gated(None, 70, 136, 264, mangle=turned)
    check_gated([0, 20, 70], 70, 136, 264, mangle=turned)
    check_act(70, 136, 264, mangle=turned)


def test_expanded_operands():
    x, w = randn(1, 64).expand(40, 64), randn(128, 64, scale=0.1)
    r = randn(1, 128, seed=1).expand(40, 128)
    y = bg.matmul_b200_act(x, w.t(), randn(1, seed=2).expand(128), r, activation="relu")
    assert torch.equal(y, y[:1].expand_as(y))
    dr, = torch.autograd.grad(
        bg.matmul_b200_act(x, w.t(), residual=(r1 := randn(1, 128).requires_grad_()).expand(40, 128)),
        r1, torch.ones(40, 128, device="cuda").bfloat16())
    assert bool((dr == 40).all())


@pytest.mark.parametrize("kernel", [0, 1, 2])
def test_padding_rows_hold_anything(kernel):
    """Rows of no expert, and their gradients, are infinities and NaN; so are the weights of
    an expert without rows."""
    capi.ffn_set_kernel(kernel)
    offsets = torch.tensor([3, 40, 40, 150], dtype=torch.int32, device="cuda")
    x, g, u, dh = randn(170, 72), randn(3, 136, 72, seed=1), randn(3, 136, 72, seed=2), randn(170, 136, seed=3)

    def run(bad):
        xs, gs, us, ds = (t.clone() for t in (x, g, u, dh))
        if bad:
            for t in (xs, ds):
                t[:3], t[150:] = float("nan"), float("inf")
            gs[1], us[1] = float("inf"), float("nan")
        xs, gs, us = (t.requires_grad_() for t in (xs, gs, us))
        h = bg.matmul_b200_gated(xs, gs.transpose(1, 2), us.transpose(1, 2), offsets)
        return (h, *torch.autograd.grad(h, (xs, gs, us), ds))
    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)


def test_values_that_are_not_finite():
    """They come out where the formula has them, and nowhere else."""
    x, w = randn(40, 64), randn(136, 64, scale=0.1)
    x[7], x[9, 3] = float("nan"), float("inf")
    y = bg.matmul_b200_act(x, w.t(), activation="relu")
    assert bool(y[7].isnan().all()) and bool(torch.isfinite(y[:7]).all())
    rest = torch.ones(40, dtype=torch.bool)
    rest[[7, 9]] = False
    assert bool(torch.isfinite(y[rest]).all())
    assert bool(((y[9] == float("inf")) == (w[:, 3] > 0)).all())
    assert bool(((y[9] == 0) == (w[:, 3] <= 0)).all())


@pytest.mark.parametrize("act", capi.ACTIVATIONS)
def test_activations_over_their_range(act):
    """act(z) and act'(z) for z from -30 to 30 and at the borders: the product with 1 is exact.

    Off by u of the value from the rounding (fp16, bf16) and 2^-16 of it from fp32 (an
    exponent of up to 30 / ln 2 rounded at 2^-24, the approximations), plus the type's
    smallest steps.  An exponential below 2^-126 is taken for zero: an error of up to 2^-126,
    which z multiplies (z Phi(z), and z phi(z) in the slope): 30 2^-126.  gelu_tanh's is
    below it from z = -10.1 on, where its slope multiplies it by 1 + |z| 2c (1 + 3 0.0447 z^2)
    = 240; further out the value itself is smaller than that: 256 2^-126."""
    lost = 256 if act == "gelu_tanh" else 30
    for dtype, u, tiny in ((torch.bfloat16, 2.0 ** -8, 2.0 ** -126), (torch.float16, 2.0 ** -11, 2.0 ** -24)):
        z = torch.linspace(-30, 30, 4001, device="cuda").to(dtype)[:, None]
        z = torch.cat([z, torch.tensor([[0.0], [-0.0], [1e-4], [-1e-4]], device="cuda").to(dtype)])
        one = torch.ones(1, 1, dtype=dtype, device="cuda")
        zg = z.clone().requires_grad_()
        y = bg.matmul_b200_act(zg, one, activation=act)
        dz, = torch.autograd.grad(y, zg, torch.ones_like(y))
        a, slope = curve(act, z.double())
        for got, want in ((y, a), (dz, slope)):
            # (a slope crosses zero: its terms are of the order of act there)
            bound = (u * 1.001 + 2.0 ** -16) * want.abs() + 2.0 ** -20 * a.abs().clamp(max=1) \
                + 2 * tiny + lost * 2.0 ** -126
            off = (got.double() - want).abs() - bound
            assert bool((off <= 0).all()), (act, dtype, float(z[off.argmax()]))


def test_bad_offsets_are_clamped_and_reported():
    x, g, u = randn(20, 64), randn(2, 64, 64, seed=1), randn(2, 64, 64, seed=2)
    for bad in ([0, 12, 30], [0, 15, 10], [-4, 3, 20]):
        a = min(max(bad[0], 0), 20)
        b = max(min(bad[1], 20), a)
        want = bg.matmul_b200_gated(x[a:b], g[0].t(), u[0].t())
        for kernel in (1, 2):
            for kind in (torch.int32, torch.int64):
                capi.ffn_set_kernel(kernel)
                off = torch.tensor(bad, dtype=kind, device="cuda")
                xg = x.clone().requires_grad_()
                y = bg.matmul_b200_gated(xg, g.transpose(1, 2), u.transpose(1, 2), off)
                torch.autograd.grad(y, xg, y)
                assert capi.device_status(True) == 0x100A
                assert float((y[a:b].double() - want.double()).norm()) <= 2.0 ** -8 * float(want.double().norm())


# ----------------------------------------------------------------- streams, graphs
STEPS = {
    # few rows, a cluster; experts; left-over tiles; streaming with divided tiles
    "cluster": (0, None, 70, 136, 2056), "stream": (1, None, 20, 136, 2056),
    "experts": (0, [0, 30, 30, 100], 100, 136, 264), "pair": (2, None, 600, 3300, 1608),
}


def step_of(name):
    kernel, offsets, rows, n, k = STEPS[name]
    bank = () if offsets is None else (len(offsets) - 1,)
    x = randn(rows, k).requires_grad_()
    g, u = (randn(*bank, n, k, seed=i, scale=k ** -0.5).requires_grad_() for i in (1, 2))
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")
    dh = randn(rows, n, seed=3)

    def step():
        capi.ffn_set_kernel(kernel)
        h = bg.matmul_b200_gated(x, g.transpose(-1, -2), u.transpose(-1, -2), off)
        # (no graph of the leaves outlives the step: torch could not capture another)
        return (h.detach(), *torch.autograd.grad(h, (x, g, u), dh))
    return x, step


@pytest.mark.parametrize("name", list(STEPS))
def test_other_stream_and_graph(name):
    x, step = step_of(name)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):   # two graphs, replayed in turn and on two streams at once
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for scale in (1.0, 2.0):
        with torch.no_grad():
            x.mul_(scale)
        want = step()
        torch.cuda.synchronize()
        for graph, _ in graphs:
            graph.replay()
        for i in range(5):
            with torch.cuda.stream(side):
                graphs[0][0].replay()
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_act_in_a_graph():
    leaves = [randn(70, 264).requires_grad_(), randn(136, 264, scale=0.06).requires_grad_(),
              randn(136, seed=1).requires_grad_(), randn(70, 136, seed=2).requires_grad_()]
    x, w, b, r = leaves
    dy = randn(70, 136, seed=3)

    def step():
        y = bg.matmul_b200_act(x, w.t(), b, r, activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    want = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_threads():
    """Three threads, each on a stream of its own, through every kernel."""
    cases = []
    for name in STEPS:
        kernel, offsets, rows, n, k = STEPS[name]
        if kernel:
            continue   # (the choice is the process's)
        cases.append(step_of(name)[1])
    cases.append(lambda: (bg.matmul_b200_act(randn(3, 512), randn(4096, 512).t(), activation="gelu"),))
    cases.append(lambda: (bg.grad_norm_b200([randn(5000), randn(7).float()]),))
    want = [c() for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                for i, c in enumerate(cases):
                    got = c()
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        bad.append(i)
    team = [threading.Thread(target=work) for _ in range(3)]
    for t in team:
        t.start()
    for t in team:
        t.join()
    assert not bad


def finish(seconds):
    """Waits for the device, but not for ever."""
    done = torch.cuda.Event()
    done.record()
    end = time.monotonic() + seconds
    while not done.query():
        if time.monotonic() > end:
            pytest.exit("a kernel does not end", returncode=1)
        time.sleep(0.001)


# clusters of single CTAs, of pairs, whole and left-over tiles
@pytest.mark.parametrize("rows,n,k,steps", [(200, 512, 512, 6000), (256, 8192, 512, 6000),
                                            (600, 1100, 640, 3000), (512, 2048, 2048, 3000)])
def test_many_steps(rows, n, k, steps):
    x, g, u = randn(rows, k), randn(n, k, scale=k ** -0.5), randn(n, k, seed=1, scale=k ** -0.5)
    with torch.no_grad():
        first = bg.matmul_b200_gated(x, g.t(), u.t())
        for i in range(steps):
            got = bg.matmul_b200_gated(x, g.t(), u.t())
            back = bg.matmul_b200_act(got, g, activation="silu")
            if i % 500 == 499:
                finish(20)
        finish(20)
    assert torch.equal(first, got) and bool(torch.isfinite(back).all())


def test_no_expert():
    x = randn(5, 16).requires_grad_()
    bank = randn(0, 16, 8).requires_grad_()
    off = torch.zeros(1, dtype=torch.int32, device="cuda")
    h = bg.matmul_b200_gated(x, bank, bank, off)
    dx, db = torch.autograd.grad(h, (x, bank), torch.ones_like(h))
    assert h.shape == (5, 8) and not h.any() and not dx.any() and db.shape == (0, 16, 8)


@pytest.mark.parametrize("m,n,k", [(40, 256, 512), (300, 260, 64), (33, 75, 128)])
def test_result_over_its_residual(m, n, k):
    """The C ABI's C may be the residual itself."""
    x, w, r = randn(m, k), randn(n, k, seed=1, scale=k ** -0.5), randn(m, n, seed=2)
    for kernel in (1, 2, 3):
        capi.ffn_set_kernel(kernel)
        want = bg.matmul_b200_act(x, w.t(), residual=r, activation="silu")
        c = r.clone()
        st = capi.lib().b200_ffn_act(x.data_ptr(), w.data_ptr(), None, c.data_ptr(), c.data_ptr(),
                                     None, m, n, k, k, k, n, n, 0, 2, capi.BF16,
                                     torch.cuda.current_stream().cuda_stream)
        assert st == capi.OK and torch.equal(c, want)


def test_rows_and_columns_past_the_result_are_left():
    """Strided results through the C ABI: what lies between rows and after them stays."""
    m, n, k = 70, 72, 128
    x, w = randn(m, k), randn(n, k, seed=1, scale=0.1)
    want = bg.matmul_b200_act(x, w.t(), activation="relu")
    for ld in (80, 75, 72):
        for kernel in (1, 2, 3):
            capi.ffn_set_kernel(kernel)
            c = torch.full((m + 3, ld), 7.0, device="cuda").bfloat16()
            z = torch.full((m + 3, 76), 5.0, device="cuda")
            st = capi.lib().b200_ffn_act(x.data_ptr(), w.data_ptr(), None, None, c.data_ptr(),
                                         z.data_ptr(), m, n, k, k, k, 0, ld, 76, 1, capi.BF16,
                                         torch.cuda.current_stream().cuda_stream)
            assert st == capi.OK
            assert float((c[:m, :n].double() - want.double()).norm()) <= 2.0 ** -8 * float(want.double().norm())
            assert bool((c[m:] == 7).all()) and bool((c[:, n:] == 7).all())
            assert bool((z[m:] == 5).all()) and bool((z[:, n:] == 5).all())


# -------------------------------------------------------------------- derivatives
def test_gradients_against_differences():
    """f = <y, c> in 64 bits moves by the gradient: central differences of h = 1/64, whose own
    error is h^2 / 6 of the third derivative (below 2^-13 of the terms' sum here)."""
    k, n, m = 16, 8, 4
    for act in ("silu", "gelu", "gelu_tanh", "sigmoid"):
        ops = [randn(m, k), randn(n, k, seed=1, scale=0.3), randn(n, k, seed=2, scale=0.3)]
        c = randn(m, n, seed=3)
        leaves = [t.clone().requires_grad_() for t in ops]
        h = bg.matmul_b200_gated(leaves[0], leaves[1].t(), leaves[2].t(), activation=act)
        grads = torch.autograd.grad(h, leaves, c)

        def f(x, g, u):
            return float((curve(act, x @ g.T)[0] * (x @ u.T) * c.double()).sum())
        step = 1.0 / 64
        for i, at in ((0, (1, 3)), (0, (3, 15)), (1, (0, 0)), (1, (7, 9)), (2, (5, 1))):
            up, down = [t.double() for t in ops], [t.double() for t in ops]
            up[i], down[i] = up[i].clone(), down[i].clone()
            up[i][at] += step
            down[i][at] -= step
            slope = (f(*up) - f(*down)) / (2 * step)
            size = float(c.double().abs().sum())
            assert abs(float(grads[i][at]) - slope) <= 2 * 2.0 ** -8 * abs(slope) + 2.0 ** -9 * size / m


def test_second_derivatives_are_refused():
    x, w, b, r = randn(4, 16), randn(8, 16), randn(8), randn(4, 8)
    for call, at in ((lambda t: bg.matmul_b200_act(t, w.t(), b, r, activation="silu"), x),
                     (lambda t: bg.matmul_b200_act(x, w.t(), t, r, activation="silu"), b),
                     (lambda t: bg.matmul_b200_gated(t, w.t(), w.t()), x),
                     (lambda t: bg.matmul_b200_gated(x, t.t(), w.t(), activation="none"), w)):
        leaf = at.clone().requires_grad_()
        out = call(leaf)
        grad, = torch.autograd.grad(out, leaf, torch.ones_like(out), create_graph=True)
        with pytest.raises(RuntimeError, match="second derivatives"):
            grad.float().sum().backward()


def test_saved_operands_are_watched():
    x, w = randn(4, 16).requires_grad_(), randn(8, 16).requires_grad_()
    y = bg.matmul_b200_gated(x, w.t(), w.t())
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_shared_and_frozen_weights():
    x, w = randn(33, 72).requires_grad_(), randn(136, 72, seed=1, scale=0.1)
    dh = randn(33, 136, seed=2)
    g, u = w.clone().requires_grad_(), w.clone().requires_grad_()
    h = bg.matmul_b200_gated(x, g.t(), u.t())
    dx, dg, du = torch.autograd.grad(h, (x, g, u), dh, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip((dx, dg, du), torch.autograd.grad(h, (x, g, u), dh)))
    only_g, = torch.autograd.grad(bg.matmul_b200_gated(x.detach(), g.t(), w.t()), g, dh)
    only_u, = torch.autograd.grad(bg.matmul_b200_gated(x.detach(), w.t(), u.t()), u, dh)
    only_x, = torch.autograd.grad(bg.matmul_b200_gated(x, w.t(), w.t()), x, dh)
    assert torch.equal(only_g, dg) and torch.equal(only_u, du) and torch.equal(only_x, dx)
    one = w.clone().requires_grad_()
    both, = torch.autograd.grad(bg.matmul_b200_gated(x, one.t(), one.t()), one, dh)
    assert torch.equal(both, dg + du)


# ----------------------------------------------------------------------- refusals
def test_refusals_on_the_device():
    x, w, b, r = randn(4, 16), randn(8, 16), randn(8), randn(4, 8)
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    bank = randn(2, 16, 8)
    bad = [
        ("inner dimensions", lambda: bg.matmul_b200_act(x, w)),
        ("dtype", lambda: bg.matmul_b200_act(x, w.t().half())),
        ("bfloat16 or float16", lambda: bg.matmul_b200_act(x.float(), w.t().float())),
        ("dtype", lambda: bg.matmul_b200_act(x, w.t(), b.float())),
        ("another device", lambda: bg.matmul_b200_act(x, w.t(), b.cpu())),
        ("bias must have shape", lambda: bg.matmul_b200_act(x, w.t(), b[:4])),
        ("residual must have shape", lambda: bg.matmul_b200_act(x, w.t(), b, r[:2])),
        ("residual must have shape", lambda: bg.matmul_b200_act(x, w.t(), b, b)),
        ("same shape", lambda: bg.matmul_b200_gated(x, w.t(), w[:4].t())),
        ("inner dimensions", lambda: bg.matmul_b200_gated(x, w, w)),
        ("dtype", lambda: bg.matmul_b200_gated(x, w.t(), w.t().half())),
        ("needs offsets", lambda: bg.matmul_b200_gated(x, bank, bank)),
        ("offsets go with a bank", lambda: bg.matmul_b200_gated(x, w.t(), w.t(), off)),
        ("offsets must have", lambda: bg.matmul_b200_gated(x, bank, bank, off[:2])),
        ("int32 or int64", lambda: bg.matmul_b200_gated(x, bank, bank, off.float())),
        ("on the operands' device", lambda: bg.matmul_b200_gated(x, bank, bank, off.cpu())),
        ("CUDA", lambda: bg.clip_grads_b200([x, x.cpu()], 1.0)),
        ("float32, bfloat16 or float16", lambda: bg.grad_norm_b200([x.double()])),
        ("share memory", lambda: bg.clip_grads_b200([x, x], 1.0)),
        ("share memory", lambda: bg.clip_grads_b200([x, x[1:]], 1.0)),
        ("share memory", lambda: bg.clip_grads_b200([x[:, :4], x[:, :4]], 1.0)),
        ("expanded", lambda: bg.clip_grads_b200([x[:1].expand(4, 16)], 1.0)),
        ("no gradient is defined", lambda: bg.clip_grads_b200([x.clone().requires_grad_()], 1.0)),
    ]
    for match, call in bad:
        with pytest.raises(RuntimeError, match=match):
            call()
    assert float(bg.grad_norm_b200([x, x])) > 0   # (read only: twice is twice)
