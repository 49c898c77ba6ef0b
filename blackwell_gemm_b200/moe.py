"""Mixture-of-experts operators: products whose weight is a bank of experts.

Rows are sorted by expert: expert e owns rows ``offsets[e] .. offsets[e+1]-1``.
``offsets`` stays on the device; no call here waits for the GPU.  Everything
runs on the current stream and is computed by libb200gemm.so
(include/b200_moe.h); there is no fallback.
"""
from __future__ import annotations

__all__ = ["matmul_b200_grouped"]


def _ext():
    from . import load
    return load()


def matmul_b200_grouped(A, B, offsets):
    """C[r] = A[r] @ B[e] for every row r of expert e; differentiable in A and B.

    A: (rows, K) bf16 or fp16 CUDA, sorted by expert.  B: (experts, K, N) of
    the same dtype, normally ``W.transpose(1, 2)`` of an (experts, N, K) bank.
    offsets: (experts + 1,) int32 or int64 on the device.  Returns (rows, N);
    rows of no expert (before offsets[0], from offsets[-1] on) are zero, in C
    and in A's gradient, and take no part in B's.  An expert may have no rows:
    its gradient is zero.  Sums are fp32, rounded once.

    The gradient of B is an (experts, K, N) view of (experts, N, K) memory, the
    layout of W.  K not a multiple of 8 (or operands otherwise not on 16-byte
    rows) costs a copy of that operand per call.  Offsets that decrease or
    leave [0, rows] are clamped and reported by ``capi.device_status``."""
    return _ext().matmul_b200_grouped(A, B, offsets)
