"""Feed-forward operators: products with the activation, gate, bias and residual
of a feed-forward layer in their epilogue, and the norm and clipping of a training
step's gradients.

Everything runs on the current stream and is computed by libb200gemm.so
(include/b200_ffn.h); there is no fallback, and no call waits for the GPU.
Gradients are first derivatives by the backward pass; forward-mode derivatives
raise at the call, second ones where they are taken.

Activations: "none", "relu", "silu" (z s(z)), "gelu" (z Phi(z)), "gelu_tanh" (its
tanh form) and "sigmoid" (s(z)), with s the logistic function and Phi the normal
distribution's.
"""
from __future__ import annotations

__all__ = ["matmul_b200_act", "matmul_b200_gated", "grad_norm_b200", "clip_grads_b200"]


_loaded = None


def _ext():
    global _loaded
    if _loaded is None:
        from . import load
        _loaded = load()
    return _loaded


def matmul_b200_act(A, B, bias=None, residual=None, *, activation: str = "none"):
    """C = act(A @ B + bias) + residual in one pass; differentiable in all four.

    A: (M, K) bf16 or fp16 CUDA; B: (K, N), normally the .T of an (N, K) weight;
    bias: (N,) or None; residual: (M, N) or None; all of A's dtype.  Sums and the
    epilogue are fp32, rounded once.

    With gradients, and an activation, its argument is kept in fp32 (4 bytes an
    element).  Its gradient is rounded to A's dtype before the products that make A's
    and B's -- in fp16 to infinity beyond 65504, where the gradients themselves might
    not be: scale the loss, or take bf16 -- and the bias' is summed before that.  What
    comes back through relu is zero up to z = 0, whatever arrives.  The gradient of B
    is a (K, N) view of (N, K) memory, the layout of the weight.  An operand whose rows
    are not on 16 bytes (K no multiple of 8) costs a copy of it per call, with gradients
    per training step."""
    return _ext().matmul_b200_act(A, B, bias, residual, activation)


def matmul_b200_gated(A, B_gate, B_up, offsets=None, *, activation: str = "silu"):
    """H = act(A @ B_gate) * (A @ B_up) in one pass; differentiable in all three.

    A: (rows, K) bf16 or fp16 CUDA; B_gate, B_up: (K, N), normally the .T of (N, K)
    weights, which may be halves of one matrix.  With offsets, banks (experts, K, N)
    of which row r takes its expert's, as in matmul_b200_grouped: rows sorted by
    expert, (experts + 1,) int32 or int64 on the device, clamped where they decrease
    or leave [0, rows]; rows of no expert are zero in H and in A's gradient and take
    no part in the weights'.  Sums and the gate are fp32, rounded once.

    With gradients both products are kept in fp32 (8 bytes an element of H), and
    their gradients, dH u act'(g) and dH act(g), are rounded to A's dtype before the
    products that follow: in fp16 to infinity beyond 65504, also where A's gradient
    would be finite (scale the loss, or take bf16).  Weight
    gradients have the layout of the (N, K) weights and share one allocation.  Operands
    that are not read as they lie cost a copy, as there."""
    return _ext().matmul_b200_gated(A, B_gate, B_up, offsets, activation)


def grad_norm_b200(grads):
    """The 2-norm of all elements of `grads` together, a 0-d float32 tensor.

    grads: tensors (at least one) of float32, bf16 and fp16 on one CUDA device, of
    any shapes, empty ones among them.  Squares are added 16 bytes of a tensor at a time
    in fp32 (in fp64 where fp32 does not hold them), those sums in fp64, in one order:
    within 2^-21 of the norm, the same bits every time."""
    return _ext().grad_norm_b200(_list(grads))


def clip_grads_b200(grads, max_norm: float):
    """Scale `grads` in place by min(1, max_norm / (norm + 1e-6)) and return their norm
    before that, a 0-d float32 tensor: grad_norm_b200 and the scaling in two launches
    (for each 320 tensors), without a wait for the device.  Where the factor is 1 (from
    a norm of max_norm - 1e-6 down) nothing is written, but for tensors with gaps between
    their elements: these go through a copy and back.  A norm that is NaN makes every
    gradient NaN, an infinite one zero, and NaN where it was infinite (every one NaN if
    max_norm is infinite too).  Elements that share memory are refused (rows, columns and
    planes that lie between one another's do not)."""
    return _ext().clip_grads_b200(_list(grads), max_norm)


def _list(grads):
    import torch
    return [grads] if isinstance(grads, torch.Tensor) else list(grads)
