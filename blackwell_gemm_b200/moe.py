"""Mixture-of-experts operators: products whose weight is a bank of experts.

Rows are sorted by expert: expert e owns rows ``offsets[e] .. offsets[e+1]-1``.
``offsets`` stays on the device; no call here waits for the GPU, but for
``pack_w4``, once per weight, to look at zero points.  Everything runs on the
current stream and is computed by libb200gemm.so (include/b200_moe.h); there is
no fallback.
Gradients are first derivatives by the backward pass; forward-mode derivatives
raise at the call, second ones where they are taken.
"""
from __future__ import annotations

from typing import NamedTuple

__all__ = ["Routing", "route_b200", "dispatch_b200", "combine_b200", "matmul_b200_grouped",
           "W4Weight", "pack_w4", "quantize_w4", "matmul_b200_w4"]


_loaded = None


def _ext():
    global _loaded
    if _loaded is None:
        from . import load
        _loaded = load()
    return _loaded


class Routing(NamedTuple):
    """Where each token's top_k slots go (route_b200)."""
    weights: "torch.Tensor"  # noqa: F821  (tokens, top_k) float32; differentiable
    experts: "torch.Tensor"  # noqa: F821  (tokens, top_k) int32, -1 at an empty slot
    rows: "torch.Tensor"     # noqa: F821  (tokens, top_k) int32, sorted row, -1 at an empty slot
    tokens: "torch.Tensor"   # noqa: F821  (tokens * top_k,) int32, -1 past the last owned row
    offsets: "torch.Tensor"  # noqa: F821  (experts + 1,) int32


def route_b200(logits, top_k: int, *, normalize: bool = True) -> Routing:
    """Each token's top_k experts, their weights, and the order by expert.

    logits: (tokens, experts) float32, bf16 or fp16 CUDA; at most 1024
    experts, top_k at most 32.  The largest logits are chosen, the lower index
    first on a tie; NaN counts as largest; an expert at -inf is closed and
    never chosen, and a token with fewer open experts than top_k has empty
    slots (expert and row -1, weight 0).  weights: the softmax over the chosen
    experts (normalize) or over all of them, in float32; differentiable in the
    logits.  Rows are sorted by expert, then token, then slot."""
    return Routing(*_ext().route_b200(logits, top_k, normalize))


def dispatch_b200(x, routing: Routing):
    """xs[row] = x[token of row]: (tokens, width) bf16 or fp16 to (tokens *
    top_k, width), sorted by expert; rows that no slot names are zero.  Slots may
    be taken out of a routing: ``routing._replace(rows=...)`` with -1 there.
    Differentiable: a token's gradient is its rows' sum, in fp32, rounded once."""
    return _ext().dispatch_b200(x, routing.rows, routing.offsets)


def combine_b200(y, routing: Routing, weights=None):
    """out[t] = sum_j weights[t, j] * y[rows[t, j]] over t's non-empty slots:
    (tokens * top_k, width) to (tokens, width), summed in fp32, rounded once.
    weights: (tokens, top_k) float32, routing.weights by default.
    Differentiable in y and the weights."""
    w = routing.weights if weights is None else weights
    return _ext().combine_b200(y, w, routing.rows, routing.offsets)


def matmul_b200_grouped(A, B, offsets):
    """C[r] = A[r] @ B[e] for every row r of expert e; differentiable in A and B.

    A: (rows, K) bf16 or fp16 CUDA, sorted by expert.  B: (experts, K, N) of
    the same dtype, normally ``W.transpose(1, 2)`` of an (experts, N, K) bank.
    offsets: (experts + 1,) int32 or int64 on the device.  Returns (rows, N);
    rows of no expert (before offsets[0], from offsets[-1] on) are zero, in C
    and in A's gradient, and take no part in B's.  An expert may have no rows:
    its gradient is zero.  Sums are fp32, rounded once.

    The gradient of B is an (experts, K, N) view of (experts, N, K) memory, the
    layout of W.  An operand that is not read as it lies costs a copy of it per
    call (with gradients: per training step): rows of W or A not on 16 bytes, as
    with K no multiple of 8, or a bank that lies as (experts, K, N).  Offsets that decrease or
    leave [0, rows] are clamped and reported by ``capi.device_status``."""
    return _ext().matmul_b200_grouped(A, B, offsets)


class W4Weight(NamedTuple):
    """4-bit weights laid out for matmul_b200_w4 (see pack_w4)."""
    data: "torch.Tensor"    # noqa: F821  packed bytes, on the device
    experts: int            # matrices; 1 and bank = False for a single one
    N: int
    K: int
    group: int
    zeros: bool
    half: bool              # fp16 scales and rows (else bf16)
    bank: bool


def pack_w4(q, scales, zeros=None) -> W4Weight:
    """Lay 4-bit weights out, once, in the order matmul_b200_w4 reads them.

    The weight of row n and column k is (q - zero) * scale, with one scale and
    one zero point per group of 32, 64 or 128 consecutive k.  q: uint8
    (N, K/2) or (experts, N, K/2), the low nibble the even k.  scales: bf16 or
    fp16, (.., N, K/group); the rows multiplied later must have the same dtype.
    zeros: uint8 0..15 of scales' shape, or None for 8 everywhere; larger ones
    raise, for which the call waits for the device."""
    bank = q.dim() == 3
    if not bank:
        if q.dim() != 2:
            raise RuntimeError("pack_w4: q must be (N, K/2) or (experts, N, K/2)")
        if scales.dim() != 2 or (zeros is not None and zeros.dim() != 2):
            raise RuntimeError("pack_w4: scales and zeros must be (N, K/group), like q")
        q, scales = q[None], scales[None]
        zeros = None if zeros is None else zeros[None]
    data = _ext().w4_pack(q, scales, zeros)
    import torch
    experts, N, K = q.shape[0], q.shape[1], 2 * q.shape[2]
    group = K // scales.shape[2] if scales.shape[2] else 128
    return W4Weight(data, experts, N, K, group, zeros is not None,
                    scales.dtype == torch.float16, bank)


def quantize_w4(w, group: int = 128):
    """(q, scales) of a bf16 or fp16 weight (.., N, K), rounded to nearest with
    symmetric scales: |w| / 7 of each group's largest.  A plain helper; any
    quantiser that yields pack_w4's operands will do."""
    *lead, n, k = w.shape
    if k % group:
        raise RuntimeError(f"quantize_w4: K = {k} is not a multiple of group = {group}")
    parts = w.float().reshape(*lead, n, k // group, group)
    scales = (parts.abs().amax(-1) / 7).to(w.dtype)
    step = scales.float().masked_fill(scales == 0, 1.0)[..., None]
    q = ((parts / step).round().clamp(-8, 7) + 8).to(dtype=_uint8()).reshape(*lead, n, k)
    return q[..., 0::2] | (q[..., 1::2] << 4), scales


def _uint8():
    import torch
    return torch.uint8


def matmul_b200_w4(A, weight: W4Weight, offsets=None):
    """C = A @ W.T for 4-bit weights; with a bank, by expert as
    matmul_b200_grouped.

    A: (rows, K) CUDA, bf16 or fp16 like the weight's scales.  offsets:
    (experts + 1,) int32 or int64 on the device, for a bank.  Returns
    (rows, N).  The weights enter unrounded, and the result is rounded once:
    either as 4-bit integers, exact, whose fp32 sums the scales multiply, or (bf16
    in groups of 32 and 64 with more than 32 rows, in a bank with more than 16 to an
    expert) as the sum of two bf16, exact for scales of 2^-120 and more.  An
    infinite scale gives a result that is not finite; where its weights differ in
    sign or are zero the first way may say inf and the second NaN.  The weights are
    read once per 8 to 256 rows of an expert.  No gradient."""
    if offsets is None and weight.bank and weight.experts != 1:
        raise RuntimeError("matmul_b200_w4: a bank of experts needs offsets")
    return _ext().w4_matmul(A, weight.data, weight.experts, weight.N, weight.K, weight.group,
                            weight.zeros, weight.half, offsets)
