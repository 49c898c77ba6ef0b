"""Gradients that share memory, with one another or within themselves, are refused wherever
their elements meet, and only there."""
import math
import random

import pytest
import torch

import blackwell_gemm_b200 as bg
from test_clip_gpu import check

pytestmark = pytest.mark.gpu


def memory():
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(8, 16, generator=g, device="cuda").bfloat16()
    y = torch.randn(4, 6, 8, generator=g, device="cuda")
    return x, y


SHARED = {
    "dense, then its columns": lambda x, y: [x, x[:, :4]],
    "columns, then what holds them": lambda x, y: [x[:, :4], x],
    "columns that cross": lambda x, y: [x[:, :4], x[:, 2:6]],
    "the same columns of later rows": lambda x, y: [x[:, :4], x[1:, :4]],
    "every second and every third row": lambda x, y: [x[::2], x[1::3]],
    "one row and columns": lambda x, y: [x[3], x[:, 5:6]],
    "planes and a point": lambda x, y: [y[:, ::2, ::2], y[1:3, 2:3, 4:6]],
    "turned": lambda x, y: [x[:, :4].t(), x[2:3, 3:9]],
    "another type": lambda x, y: [x.view(torch.float32)[:, :2], x[:, 3:8]],
    "half of an element": lambda x, y: [y[:, ::2, ::2], y.view(torch.bfloat16)[1:2, 2:3, 1:2]],
    "a diagonal": lambda x, y: [x.as_strided((8,), (17,)), x[:, 4:8]],
    "windows of one tensor": lambda x, y: [x.as_strided((5, 8), (4, 1))],
    "a row and the next, shifted": lambda x, y: [y, x.as_strided((3, 3), (1, 1))],
    "two dimensions of one stride": lambda x, y: [x.as_strided((2, 2, 3), (20, 20, 3))],
    "strides that meet": lambda x, y: [x.as_strided((4, 5), (6, 4))],
    "third among others": lambda x, y: [x[:, :4], x[:, 8:], y, x[5:6, 3:5]],
}
APART = {
    "columns": lambda x, y: [x[:, :4], x[:, 4:8], x[:, 12:]],
    "rows in turn": lambda x, y: [x[::2], x[1::2]],
    "columns in turn": lambda x, y: [x[:, ::2], x[:, 1::2]],
    "planes": lambda x, y: [y[:, ::2, ::2], y[:, 1::2, ::2], y[:, :, 1::2]],
    "between the rows": lambda x, y: [x[:, :4], x[0, 4:16], x[1, 4:16]],
    "another type": lambda x, y: [x.view(torch.float32)[:, :2], x[:, 4:8]],
    "a diagonal": lambda x, y: [x.as_strided((4,), (17,)), x[:, 4:8]],
    "strides that do not meet": lambda x, y: [x.as_strided((2, 4), (9, 6))],
    "strides out of order": lambda x, y: [x.as_strided((2, 3, 4), (3, 40, 7))],
    "empty": lambda x, y: [x[:, :4], x[:, 2:2], x[3:3]],
}


@pytest.mark.parametrize("name", list(SHARED))
def test_shared(name):
    grads = SHARED[name](*memory())
    keep = [g.clone() for g in grads]
    for order in (grads, grads[::-1]):
        with pytest.raises(RuntimeError, match="share memory"):
            bg.clip_grads_b200(order, 0.5)
    assert all(torch.equal(g, k) for g, k in zip(grads, keep))
    assert float(bg.grad_norm_b200(grads)) > 0   # (read only)


@pytest.mark.parametrize("name", list(APART))
def test_apart(name):
    x, y = memory()
    for order in (1, -1):
        check(APART[name](x, y)[::order], 0.5)


def test_many_columns():
    """All extents cross; no element does."""
    x = torch.randn(40, 300, device="cuda")
    check([x[:, i:i + 1] for i in range(300)], 0.5)
    with pytest.raises(RuntimeError, match="share memory"):
        bg.clip_grads_b200([x[:, i:i + 1] for i in range(300)] + [x[7:9, 255:257]], 0.5)


def test_against_enumeration():
    """Views of one buffer with any strides, of both element sizes: refused exactly where two
    elements have a byte in common."""
    r = random.Random(0)
    wide = torch.randn(200, device="cuda")
    buffers = {4: wide, 2: wide.view(torch.bfloat16)}
    seen = [0, 0]
    for _ in range(600):
        views, taken, met = [], set(), False
        for _ in range(r.randint(1, 3)):
            size = r.choice([2, 4])
            flat = buffers[size]
            shape = [r.randint(1, 4) for _ in range(r.randint(1, 3))]
            strides = [r.choice([1, 2, 3, 5, 8, 12, 16, 20]) for _ in shape]
            start = r.randint(0, 400 // size)
            at = [start]
            for n, s in zip(shape, strides):
                at = [a + i * s for a in at for i in range(n)]
            assert max(at) < flat.numel()
            for a in at:
                mine = {a * size + b for b in range(size)}
                met |= bool(mine & taken)
                taken |= mine
            views.append(flat.as_strided(shape, strides, start))
        seen[met] += 1
        if met:
            with pytest.raises(RuntimeError, match="share memory"):
                bg.clip_grads_b200(views, math.inf)
        else:
            bg.clip_grads_b200(views, math.inf)
    assert min(seen) > 100, seen
