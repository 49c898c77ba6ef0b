"""CTA pairs that start beside the end of another kernel.

A pair's tensor memory may be asked for only once both CTAs run.  Pair kernels
that asked earlier stopped for good, a pair in some 100,000, in streams of
training steps whose launches follow one another closely.  Here: enough steps
that it showed many times over."""
import time

import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi

pytestmark = pytest.mark.gpu


def finish(seconds):
    """Waits for the device, but not for ever."""
    done = torch.cuda.Event()
    done.record()
    end = time.monotonic() + seconds
    while not done.query():
        if time.monotonic() > end:
            pytest.exit("a kernel does not end", returncode=1)
        time.sleep(0.001)


@pytest.mark.parametrize("rows,experts,n,k,dtype,steps", [
    (2364, 16, 4864, 1058, torch.float16, 8000), (2048, 16, 512, 512, torch.bfloat16, 10000)])
def test_many_training_steps(rows, experts, n, k, dtype, steps):
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(rows, k, generator=g, device="cuda").to(dtype).requires_grad_()
    w = (torch.randn(experts, n, k, generator=g, device="cuda") * k ** -0.5).to(dtype).requires_grad_()
    dy = torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    off = (torch.arange(experts + 1, device="cuda") * rows // experts).int()

    def step():
        y = bg.matmul_b200_grouped(x, w.transpose(1, 2), off)
        return (y, *torch.autograd.grad(y, (x, w), dy))
    first = step()
    for i in range(steps):
        got = step()
        if i % 500 == 499:
            finish(20)
    finish(20)
    assert all(torch.equal(a, b) for a, b in zip(first, got))
    assert capi.device_status(True) == 0


def test_many_products_in_a_row():
    a = torch.randint(-2, 3, (512, 512), device="cuda").bfloat16()
    b = torch.randint(-2, 3, (768, 512), device="cuda").bfloat16()
    want = (a.double() @ b.double().T).bfloat16()
    for i in range(20000):
        c = bg.matmul_b200(a, b.t())
        if i % 2000 == 1999:
            finish(20)
    finish(20)
    assert torch.equal(c, want)
    assert capi.device_status(True) == 0
