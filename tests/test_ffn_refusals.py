"""What the feed-forward operators refuse, checked before any device is touched
(so this runs without a GPU)."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwad

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi

FAKE = 0x7F0000000000  # never dereferenced: validation fails or returns first
INT_MAX = 2 ** 31 - 1
BAD, ALIGN, LARGE, OK = (capi.ERR_INVALID_ARGUMENT, capi.ERR_ALIGNMENT, capi.ERR_TOO_LARGE, capi.OK)


def act(a=FAKE, w=FAKE, bias=FAKE, r=FAKE, c=FAKE, z=FAKE, rows=8, n=8, k=8, lda=8, ldw=8, ldr=8,
        ldc=8, ldz=8, act=2, dtype=capi.BF16):
    return capi.lib().b200_ffn_act(a, w, bias, r, c, z, rows, n, k, lda, ldw, ldr, ldc, ldz, act,
                                   dtype, None)


@pytest.mark.parametrize("change,expect", [
    (dict(rows=-1), BAD), (dict(n=-1), BAD), (dict(k=-1), BAD), (dict(dtype=2), BAD),
    (dict(act=-1), BAD), (dict(act=6), BAD), (dict(a=0), BAD), (dict(w=0), BAD), (dict(c=0), BAD),
    (dict(k=16, ldw=16), BAD), (dict(k=16, lda=16), BAD), (dict(n=16, ldr=16, ldz=16), BAD),
    (dict(n=16, ldc=16, ldz=16), BAD), (dict(n=16, ldc=16, ldr=16), BAD),
    (dict(a=FAKE + 2), ALIGN), (dict(w=FAKE + 8), ALIGN), (dict(lda=12), ALIGN),
    (dict(ldw=12), ALIGN), (dict(c=FAKE + 1), ALIGN), (dict(r=FAKE + 1), ALIGN),
    (dict(bias=FAKE + 1), ALIGN), (dict(z=FAKE + 8), ALIGN), (dict(ldz=10), ALIGN),
    (dict(rows=INT_MAX), LARGE), (dict(n=INT_MAX - 7, ldc=INT_MAX, ldr=INT_MAX, ldz=INT_MAX - 3), LARGE),
    (dict(rows=2 ** 30, n=2 ** 30, ldc=2 ** 30, ldr=2 ** 30, ldz=2 ** 30), LARGE),
    (dict(rows=0, a=0, w=0, c=0, r=0, z=0), OK), (dict(n=0, a=0, w=0, c=0, r=0, z=0, bias=0), OK),
])
def test_act_c_abi(change, expect):
    assert act(**change) == expect


def gated(a=FAKE, g=FAKE, u=FAKE, off=FAKE, h=FAKE, z=FAKE, rows=8, experts=2, n=8, k=8, lda=8,
          ldg=8, sg=64, ldu=8, su=64, ldh=8, ldz=8, act=2, dtype=capi.BF16):
    return capi.lib().b200_ffn_gated(a, g, u, off, h, z, rows, experts, n, k, lda, ldg, sg, ldu, su,
                                     ldh, ldz, act, dtype, None)


@pytest.mark.parametrize("change,expect", [
    (dict(rows=-1), BAD), (dict(experts=-1), BAD), (dict(n=-1), BAD), (dict(k=-1), BAD),
    (dict(dtype=2), BAD), (dict(act=7), BAD), (dict(a=0), BAD), (dict(g=0), BAD), (dict(u=0), BAD),
    (dict(h=0), BAD), (dict(off=0), BAD), (dict(off=0, experts=0), BAD), (dict(ldg=0), BAD),
    (dict(sg=56), BAD), (dict(su=56), BAD), (dict(k=16, ldg=16, ldu=16, sg=128, su=128), BAD),
    (dict(n=16, sg=128, su=128, ldz=16), BAD), (dict(n=16, sg=128, su=128, ldh=16), BAD),
    (dict(a=FAKE + 2), ALIGN), (dict(g=FAKE + 2), ALIGN), (dict(u=FAKE + 2), ALIGN),
    (dict(off=FAKE + 2), ALIGN), (dict(ldu=12, su=96), ALIGN), (dict(sg=68), ALIGN),
    (dict(h=FAKE + 1), ALIGN), (dict(z=FAKE + 4), ALIGN), (dict(ldz=9), ALIGN),
    (dict(experts=1025), LARGE), (dict(rows=INT_MAX), LARGE),
    (dict(rows=2 ** 30, n=2 ** 30, sg=2 ** 33, su=2 ** 33, ldh=2 ** 30, ldz=2 ** 30), LARGE),
    (dict(rows=0, a=0, g=0, u=0, h=0, z=0), OK), (dict(n=0, g=0, u=0, h=0, z=0), OK),
])
def test_gated_c_abi(change, expect):
    assert gated(**change) == expect


def changed(function, good, changes):
    for change, expect in changes:
        args = list(good)
        for at, value in change.items():
            args[at] = value
        assert function(*args) == expect, (change, expect)


def test_gradients_c_abi():
    lib = capi.lib()
    changed(lib.b200_ffn_act_grad, [FAKE, FAKE, FAKE, FAKE, 8, 8, 8, 8, 8, 2, 0, None], [
        ({0: 0}, BAD), ({1: 0}, BAD), ({4: -1}, BAD), ({5: -1}, BAD), ({6: 4}, BAD), ({7: 4}, BAD),
        ({8: 4}, BAD), ({9: 9}, BAD), ({10: 2}, BAD), ({0: FAKE + 2}, ALIGN), ({1: FAKE + 4}, ALIGN),
        ({2: FAKE + 8}, ALIGN), ({3: FAKE + 1}, ALIGN), ({6: 12}, ALIGN), ({8: 12}, ALIGN),
        ({4: INT_MAX}, LARGE), ({2: 0, 3: 0}, OK), ({5: 0, 0: 0}, OK), ({4: 0, 3: 0}, OK)])
    changed(lib.b200_ffn_gated_grad,
            [FAKE, FAKE, FAKE, FAKE, 8, 2, 8, 8, 8, 8, 2, 0, None], [
                ({0: 0}, BAD), ({1: 0}, BAD), ({2: 0}, BAD), ({3: 0}, BAD), ({4: -1}, BAD),
                ({7: 4}, BAD), ({8: 4}, BAD), ({9: 4}, BAD), ({10: -1}, BAD), ({2: FAKE + 1}, ALIGN),
                ({0: FAKE + 2}, ALIGN), ({1: FAKE + 4}, ALIGN), ({3: FAKE + 8}, ALIGN),
                ({9: 12}, ALIGN), ({5: 1025}, LARGE), ({4: 0, 0: 0, 1: 0, 3: 0}, OK)])
    changed(lib.b200_ffn_da,
            [FAKE, FAKE, FAKE, FAKE, FAKE, 2, 8, 2, 8, 8, 8, 8, 64, 8, 64, 8, 0, None], [
                ({5: 3}, BAD), ({5: 0}, BAD), ({0: 0}, BAD), ({1: 0}, BAD), ({2: 0}, BAD), ({3: 0}, BAD),
                ({4: 0}, BAD), ({10: 4}, BAD), ({11: 4}, BAD), ({12: 56}, BAD), ({15: 4}, BAD),
                ({16: 2}, BAD), ({0: FAKE + 2}, ALIGN), ({2: FAKE + 2}, ALIGN), ({4: FAKE + 1}, ALIGN),
                ({13: 12, 14: 96}, ALIGN), ({7: 1025}, LARGE), ({6: 0, 0: 0, 1: 0, 2: 0, 4: 0}, OK)])
    changed(lib.b200_ffn_dw, [FAKE, FAKE, FAKE, FAKE, 2, 8, 2, 8, 8, 8, 8, 0, None], [
        ({4: 0}, BAD), ({0: 0}, BAD), ({1: 0}, BAD), ({2: 0}, BAD), ({3: 0}, BAD), ({9: 4}, BAD),
        ({10: 4}, BAD), ({11: 3}, BAD), ({0: FAKE + 2}, ALIGN), ({1: FAKE + 2}, ALIGN),
        ({3: FAKE + 1}, ALIGN), ({9: 12}, ALIGN), ({6: 1025}, LARGE),
        ({7: 2 ** 30, 8: 2 ** 30, 9: 2 ** 30, 10: 2 ** 30}, LARGE), ({7: 0, 0: 0, 3: 0}, OK)])
    assert lib.b200_ffn_set_kernel(4) == BAD and lib.b200_ffn_set_kernel(-1) == BAD


def test_norm_c_abi():
    lib = capi.lib()

    def call(data=FAKE, count=8, type=capi.BF16, n=1, norm=FAKE, most=1.0):
        t = (capi.Tensor * 1)(capi.Tensor(data, count, type))
        return lib.b200_grad_norm(t, n, norm, None), lib.b200_clip_grads(t, n, most, norm, None)
    assert call(data=0) == (BAD, BAD)
    assert call(count=-1) == (BAD, BAD)
    assert call(type=3) == (BAD, BAD)
    assert call(n=-1) == (BAD, BAD)
    assert call(norm=0) == (BAD, BAD)
    assert call(norm=FAKE + 2) == (ALIGN, ALIGN)
    assert call(data=FAKE + 1) == (ALIGN, ALIGN)
    assert call(data=FAKE + 2, type=capi.FP32) == (ALIGN, ALIGN)
    assert call(most=-1.0, data=0)[1] == BAD and call(most=float("nan"), n=0)[1] == BAD
    null = ctypes.POINTER(capi.Tensor)()
    assert lib.b200_grad_norm(null, 1, FAKE, None) == BAD


def calls():
    x, w, r, b = (torch.zeros(4, 8).bfloat16(), torch.zeros(8, 16).bfloat16(),
                  torch.zeros(4, 16).bfloat16(), torch.zeros(16).bfloat16())
    return [("A", lambda t: bg.matmul_b200_act(t, w, b, r), x),
            ("B", lambda t: bg.matmul_b200_act(x, t, b, r), w),
            ("bias", lambda t: bg.matmul_b200_act(x, w, t, r), b),
            ("residual", lambda t: bg.matmul_b200_act(x, w, b, t), r),
            ("gated A", lambda t: bg.matmul_b200_gated(t, w, w), x),
            ("gate", lambda t: bg.matmul_b200_gated(x, t, w), w),
            ("up", lambda t: bg.matmul_b200_gated(x, w, t), w),
            ("norm", lambda t: bg.grad_norm_b200([b, t]), x),
            ("clip", lambda t: bg.clip_grads_b200([b, t], 1.0), x)]


def test_tangents_and_host_tensors_are_refused():
    for name, call, at in calls():
        with pytest.raises(RuntimeError, match="CUDA"):
            call(at)
        with fwad.dual_level():
            dual = fwad.make_dual(at, torch.ones_like(at))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)


def test_ranks_and_names():
    x, w = torch.zeros(4, 8).bfloat16(), torch.zeros(8, 16).bfloat16()
    with pytest.raises(RuntimeError, match="must be"):
        bg.matmul_b200_act(x[0], w)
    with pytest.raises(RuntimeError, match="must be"):
        bg.matmul_b200_gated(x, w[0], w[0])
    for call in (lambda: bg.matmul_b200_act(x, w, activation="swish"),
                 lambda: bg.matmul_b200_gated(x, w, w, activation="SiLU")):
        with pytest.raises(RuntimeError, match="unknown activation"):
            call()
    with pytest.raises(RuntimeError, match="at least one"):
        bg.grad_norm_b200([])
    with pytest.raises(RuntimeError, match="at least one"):
        bg.clip_grads_b200([], 1.0)
    for most in (-1.0, float("nan")):
        with pytest.raises(RuntimeError, match="max_norm"):
            bg.clip_grads_b200([x], most)
