"""Derivatives the mixture-of-experts operators do not have are refused, not
taken for zero: forward-mode ones at the call, second ones where they are
asked for."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

import blackwell_gemm_b200 as bg


def operands(device):
    g = torch.Generator(device=device).manual_seed(0)

    def randn(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g, device=device).to(dtype)
    off = torch.tensor([0, 3, 8], dtype=torch.int32, device=device)
    rows = torch.arange(8, dtype=torch.int32, device=device).reshape(4, 2)
    routing = bg.Routing(torch.ones(4, 2, device=device), rows, rows, rows.flatten(), off)
    weight = bg.W4Weight(torch.zeros(0, dtype=torch.uint8, device=device), 1, 0, 64, 64, False, False,
                         False)
    return randn, off, routing, weight


def calls(device):
    """(name, function, the operands it may have a tangent in)"""
    randn, off, routing, weight = operands(device)
    x, w, y = randn(8, 64), randn(2, 64, 32), randn(8, 16)
    return [("grouped A", lambda t: bg.matmul_b200_grouped(t, w, off), x),
            ("grouped B", lambda t: bg.matmul_b200_grouped(x, t, off), w),
            ("route", lambda t: bg.route_b200(t, 2)[0], randn(4, 8, dtype=torch.float32)),
            ("dispatch", lambda t: bg.dispatch_b200(t, routing), randn(4, 16)),
            ("combine y", lambda t: bg.combine_b200(t, routing), y),
            ("combine weights", lambda t: bg.combine_b200(y, routing, t),
             torch.ones(4, 2, device=device)),
            ("w4", lambda t: bg.matmul_b200_w4(t, weight), x)]


def tangents(device):
    for name, call, at in calls(device):
        with fwad.dual_level():
            dual = fwad.make_dual(at, torch.ones_like(at))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)


def test_tangents_are_refused():
    tangents("cpu")


@pytest.mark.gpu
def test_tangents_are_refused_on_the_device():
    tangents("cuda")
    for name, call, at in calls("cuda"):
        call(at)
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (at,), (torch.ones_like(at),))


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    for name, call, at in calls("cuda"):
        if name == "w4":
            continue
        leaf = at.clone().requires_grad_()
        out = call(leaf)
        seed = torch.randn_like(out)
        plain, = torch.autograd.grad(out, leaf, seed)
        out = call(leaf)
        got, = torch.autograd.grad(out, leaf, seed.clone().requires_grad_(), create_graph=True)
        assert torch.equal(got, plain) and got.requires_grad
        with pytest.raises(RuntimeError, match="twice"):
            got.float().sum().backward()


@pytest.mark.gpu
def test_second_derivatives_through_the_other_operand():
    randn, off, routing, _ = operands("cuda")
    x, w = randn(8, 64).requires_grad_(), randn(2, 64, 32).requires_grad_()
    y = bg.matmul_b200_grouped(x, w, off)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)   # depends on w
    with pytest.raises(RuntimeError, match="twice"):
        dx.float().sum().backward()
    y, weights = randn(8, 16).requires_grad_(), torch.ones(4, 2, device="cuda", requires_grad=True)
    out = bg.combine_b200(y, routing, weights)
    dy, dw = torch.autograd.grad(out, (y, weights), torch.ones_like(out), create_graph=True)
    for g in (dy, dw):
        with pytest.raises(RuntimeError, match="twice"):
            g.float().sum().backward(retain_graph=True)
    # the softmax's gradient depends on the logits themselves
    logits = randn(4, 8, dtype=torch.float32).requires_grad_()
    r = bg.route_b200(logits, 2)
    d, = torch.autograd.grad(r.weights, logits, torch.randn(4, 2, device="cuda"), create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        d.sum().backward()


@pytest.mark.gpu
def test_constant_gradients_need_no_graph():
    # linear in the one operand that is differentiated: a recorded pass holds a constant
    randn, off, routing, _ = operands("cuda")
    x, w = randn(8, 64).requires_grad_(), randn(2, 64, 32)
    y = bg.matmul_b200_grouped(x, w, off)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    assert not dx.requires_grad
    x = randn(4, 16).requires_grad_()
    xs = bg.dispatch_b200(x, routing)
    dx, = torch.autograd.grad(xs, x, torch.ones_like(xs), create_graph=True)
    assert not dx.requires_grad and bool((dx == 2).all())
