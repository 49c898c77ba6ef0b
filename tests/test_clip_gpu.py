"""The norm of many gradients and their clipping, against 64 bits.

Tolerances.  Eight squares are added in fp32: each sum is off by at most 8 2^-24 of itself
(all terms are positive), the rest is fp64; the root halves that, and the result is rounded to
fp32: 5 2^-24 in all, taken as 2^-21.  The scale is that far off and is rounded (2^-24), a
product is rounded in fp32 (2^-24) and to the gradient's type (u)."""
import math

import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
OFF = 2.0 ** -21
MIXED = (torch.bfloat16, torch.float32, torch.float16)


def tensors(sizes, types=MIXED, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, generator=g, device="cuda") * scale).to(types[i % len(types)])
            for i, n in enumerate(sizes)]


def norm_of(grads):
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))


def check(grads, max_norm=1.0):
    before = [g.detach().clone() for g in grads]
    want = norm_of(grads)
    n0 = bg.grad_norm_b200(grads)
    assert n0.shape == () and n0.dtype == torch.float32
    norm = bg.clip_grads_b200(grads, max_norm)
    assert torch.equal(norm, n0)
    assert abs(float(norm) - want) <= OFF * want
    c = min(1.0, max_norm / (want + 1e-6))
    for g, b in zip(grads, before):
        if c == 1.0:
            assert torch.equal(g, b)
            continue
        w = b.double() * c
        bound = w.abs() * (U[g.dtype] * 1.001 + OFF + 2.0 ** -22) + TINY[g.dtype]
        assert bool(((g.double() - w).abs() <= bound).all())
    return norm


@pytest.mark.parametrize("sizes", [(1,), (7,), (8,), (9, 1, 3), (0, 5, 0), (16384,), (16385, 16383),
                                   (100000, 3, 65536, 1), (3000001,)])
@pytest.mark.parametrize("types", [MIXED, (torch.float32,), (torch.bfloat16,), (torch.float16,)])
def test_sizes(sizes, types):
    check(tensors(sizes, types))
    check(tensors(sizes, types), 1e9)


def test_tables():
    """More tensors than a launch's table holds."""
    for count in (319, 320, 321, 1000):
        check(tensors([1 + i % 70 for i in range(count)]))


def test_starts():
    """Views that begin on any element, one after another in one buffer."""
    for dtype in MIXED:
        flat = tensors([60000], (dtype,))[0]
        keep = flat.clone()
        views, at = [], 1
        for n in (1, 3, 17, 255, 16384, 16390, 1001):
            views.append(flat[at:at + n])
            at += n + 2
        gaps = torch.ones(60000, dtype=torch.bool, device="cuda")
        for v in views:
            start = v.storage_offset()
            gaps[start:start + v.numel()] = False
        check(views)
        assert torch.equal(flat[gaps], keep[gaps])


def test_shapes_and_strides():
    g = torch.randn(40, 64, 33, device="cuda")
    check([g.transpose(1, 2), torch.randn(5, 6, device="cuda").t()])   # dense, any order
    wide = torch.randn(64, 96, device="cuda").bfloat16()
    keep = wide.clone()
    check([wide[:, :40], wide[:, 50:], torch.randn(3, device="cuda")])  # interleaved columns
    assert torch.equal(wide[:, 40:50], keep[:, 40:50])
    check([torch.randn((), device="cuda")])


# squares that fp32 does not hold, or holds only in part; a tensor of zeros
@pytest.mark.parametrize("scale", [1e25, 1e19, 1e-15, 1e-21, 1e-25])
def test_far_values(scale):
    check(tensors([5000, 1], (torch.float32, torch.bfloat16), scale=scale), 0.5 * scale)
    mixed = tensors([5000], (torch.float32,), scale=scale) + tensors([5000], (torch.float32,))
    check(mixed, 0.5)


def test_zeros():
    z = [torch.zeros(1000, device="cuda"), torch.zeros(3, device="cuda").half()]
    assert float(check(z)) == 0.0
    assert float(bg.clip_grads_b200(z, 0.0)) == 0.0 and not any(t.any() for t in z)


def test_not_finite():
    g = tensors([100, 20000])
    g[1][777] = math.nan
    assert math.isnan(float(bg.clip_grads_b200(g, 1.0)))
    assert all(bool(t.isnan().all()) for t in g)
    g = tensors([100, 20000])
    g[1][777] = -math.inf
    assert float(bg.clip_grads_b200(g, 1.0)) == math.inf
    assert bool(g[1][777].isnan()) and not g[0].any() and int(g[1].isnan().sum()) == 1
    assert not g[1].nan_to_num().any()
    g = tensors([100])
    keep = g[0].clone()
    bg.clip_grads_b200(g, math.inf)
    assert torch.equal(g[0], keep)
    bg.clip_grads_b200(g, 0.0)
    assert not g[0].any()


def test_same_bits():
    a = tensors([200000, 77, 500001])
    norms = {float(bg.grad_norm_b200(a)) for _ in range(5)}
    assert len(norms) == 1


def test_versions():
    """What autograd saved of a gradient is no longer that."""
    x = torch.randn(8, device="cuda", requires_grad=True)
    w = torch.randn(8, device="cuda")
    y = (x * w).sum()
    bg.clip_grads_b200([w], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_training_gradients():
    p = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in ((300, 40), (40,), ())]
    q = [torch.nn.Parameter(t.detach().clone()) for t in p]
    for ps in (p, q):
        sum((t * (i + 2) ** 2).square().sum() for i, t in enumerate(ps)).backward()
    want = torch.nn.utils.clip_grad_norm_(q, 1.0)
    got = bg.clip_grads_b200([t.grad for t in p], 1.0)
    assert abs(float(got) - float(want)) <= 1e-5 * float(want)
    for a, b in zip(p, q):
        assert torch.allclose(a.grad, b.grad, rtol=1e-5, atol=0)


def test_graph_and_streams():
    g = tensors([30000, 5, 700])
    keep = [t.clone() for t in g]
    bg.clip_grads_b200(g, 1.0)
    want = [t.clone() for t in g]
    side = torch.cuda.Stream()
    for t, k in zip(g, keep):
        t.copy_(k)
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        norm = bg.clip_grads_b200(g, 1.0)
    for _ in range(3):
        for t, k in zip(g, keep):
            t.copy_(k)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(g, want))
        assert abs(float(norm) - norm_of(keep)) <= OFF * norm_of(keep)
