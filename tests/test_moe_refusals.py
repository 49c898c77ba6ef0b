"""What the mixture-of-experts operators refuse, checked before any device is
touched (so this runs without a GPU)."""
import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi

FAKE = 0x7F0000000000  # never dereferenced: validation fails or returns first
INT_MAX = 2 ** 31 - 1


def grouped(a=FAKE, b=FAKE, c=FAKE, off=FAKE, rows=8, experts=2, n=8, k=8, lda=8, ldb=8,
            stride=64, ldc=8, dtype=capi.BF16):
    return capi.lib().b200_grouped_gemm(a, b, c, off, rows, experts, n, k, lda, ldb, stride, ldc,
                                        dtype, None)


@pytest.mark.parametrize("change,expect", [
    (dict(rows=-1), capi.ERR_INVALID_ARGUMENT),
    (dict(experts=-1), capi.ERR_INVALID_ARGUMENT),
    (dict(n=-1), capi.ERR_INVALID_ARGUMENT),
    (dict(k=-1), capi.ERR_INVALID_ARGUMENT),
    (dict(dtype=2), capi.ERR_INVALID_ARGUMENT),
    (dict(a=0), capi.ERR_INVALID_ARGUMENT),
    (dict(b=0), capi.ERR_INVALID_ARGUMENT),
    (dict(c=0), capi.ERR_INVALID_ARGUMENT),
    (dict(off=0), capi.ERR_INVALID_ARGUMENT),
    (dict(k=16, ldb=16, stride=128), capi.ERR_INVALID_ARGUMENT),    # lda < K
    (dict(k=16, lda=16, stride=128), capi.ERR_INVALID_ARGUMENT),    # ldb < K
    (dict(n=16, stride=128), capi.ERR_INVALID_ARGUMENT),            # ldc < N
    (dict(stride=56), capi.ERR_INVALID_ARGUMENT),                   # matrices overlap
    (dict(a=FAKE + 2), capi.ERR_ALIGNMENT),
    (dict(b=FAKE + 8), capi.ERR_ALIGNMENT),
    (dict(c=FAKE + 1), capi.ERR_ALIGNMENT),                         # (written: any 2 bytes)
    (dict(off=FAKE + 2), capi.ERR_ALIGNMENT),
    (dict(lda=12), capi.ERR_ALIGNMENT),
    (dict(ldb=12, stride=96), capi.ERR_ALIGNMENT),
    (dict(stride=68), capi.ERR_ALIGNMENT),
    (dict(experts=1025), capi.ERR_TOO_LARGE),
    (dict(rows=INT_MAX, n=INT_MAX, ldc=INT_MAX - 7, stride=2 ** 40), capi.ERR_INVALID_ARGUMENT),
    (dict(rows=2 ** 30, n=2 ** 30, ldc=2 ** 30, stride=2 ** 33), capi.ERR_TOO_LARGE),
    (dict(rows=0, a=0, c=0), capi.OK),
    (dict(n=0, b=0, c=0), capi.OK),
])
def test_grouped_c_abi(change, expect):
    assert grouped(**change) == expect


def test_grouped_gradients_c_abi():
    lib = capi.lib()
    da = lambda **k: lib.b200_grouped_gemm_da(*_args(k, ldc=8, ldb=8, stride=64, last=8))  # noqa: E731
    assert da(rows=-1) == capi.ERR_INVALID_ARGUMENT
    assert da(p0=FAKE + 2) == capi.ERR_ALIGNMENT
    assert da(rows=0) == capi.OK
    args = [FAKE, FAKE, FAKE, FAKE, 8, 2, 8, 8, 8, 8, 8, 64, capi.BF16, None]
    for at, value, expect in [(0, 0, capi.ERR_INVALID_ARGUMENT), (2, FAKE + 1, capi.ERR_ALIGNMENT),
                              (1, FAKE + 4, capi.ERR_ALIGNMENT),
                              (8, 4, capi.ERR_INVALID_ARGUMENT), (11, 8, capi.ERR_INVALID_ARGUMENT),
                              (5, 0, capi.OK), (6, 0, capi.OK), (12, 7, capi.ERR_INVALID_ARGUMENT)]:
        changed = list(args)
        changed[at] = value
        assert lib.b200_grouped_gemm_db(*changed) == expect, (at, value)
    for bad in (-1, 3):
        with pytest.raises(capi.GemmError):
            capi.grouped_set_kernel(bad)


def _args(k, ldc, ldb, stride, last):
    return [k.get("p0", FAKE), FAKE, FAKE, FAKE, k.get("rows", 8), 2, 8, 8, ldc, ldb, stride, last,
            capi.BF16, None]


def test_grouped_torch_checks():
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    w = torch.zeros(2, 8, 8, dtype=torch.bfloat16)
    off = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        bg.matmul_b200_grouped(x, w, off)
    with pytest.raises(RuntimeError, match="experts, K, N"):
        bg.matmul_b200_grouped(x, w[0], off)
    with pytest.raises(RuntimeError, match="rows, K"):
        bg.matmul_b200_grouped(x[0], w, off)


def w4(a=FAKE, p=FAKE, c=FAKE, off=0, rows=8, experts=1, n=8, k=64, group=64, zeros=0, lda=64,
       ldc=8, dtype=capi.BF16):
    return capi.lib().b200_w4_gemm(a, p, c, off, rows, experts, n, k, group, zeros, lda, ldc,
                                   dtype, None)


@pytest.mark.parametrize("change,expect", [
    (dict(rows=-1), capi.ERR_INVALID_ARGUMENT),
    (dict(experts=-1), capi.ERR_INVALID_ARGUMENT),
    (dict(experts=2), capi.ERR_INVALID_ARGUMENT),          # a bank without offsets
    (dict(group=16), capi.ERR_INVALID_ARGUMENT),
    (dict(k=96, lda=96), capi.ERR_INVALID_ARGUMENT),       # not whole groups
    (dict(dtype=5), capi.ERR_INVALID_ARGUMENT),
    (dict(a=0), capi.ERR_INVALID_ARGUMENT),
    (dict(p=0), capi.ERR_INVALID_ARGUMENT),
    (dict(c=0), capi.ERR_INVALID_ARGUMENT),
    (dict(lda=56), capi.ERR_INVALID_ARGUMENT),
    (dict(n=16), capi.ERR_INVALID_ARGUMENT),               # ldc < N
    (dict(lda=68), capi.ERR_ALIGNMENT),
    (dict(a=FAKE + 2), capi.ERR_ALIGNMENT),
    (dict(p=FAKE + 8), capi.ERR_ALIGNMENT),
    (dict(c=FAKE + 1), capi.ERR_ALIGNMENT),                # (written: any 2 bytes)
    (dict(off=FAKE + 1, experts=2), capi.ERR_ALIGNMENT),
    (dict(experts=1025, off=FAKE), capi.ERR_TOO_LARGE),
    (dict(n=INT_MAX - 7, ldc=INT_MAX - 7, rows=INT_MAX), capi.ERR_TOO_LARGE),
    (dict(rows=0, a=0, c=0), capi.OK),
    (dict(n=0, c=0), capi.OK),
])
def test_w4_c_abi(change, expect):
    assert w4(**change) == expect


def test_w4_packed_bytes():
    import ctypes
    size = ctypes.c_size_t(0)
    lib = capi.lib()
    for args, want in [((1, 128, 128, 128, 0), 8192 + 256), ((1, 1, 32, 32, 1), 8192 + 1024 + 512),
                       ((3, 129, 192, 64, 0), 3 * 2 * 2 * (8192 + 512)), ((0, 8, 64, 64, 0), 0),
                       ((1, 0, 64, 64, 0), 0)]:
        assert lib.b200_w4_packed_bytes(*args, ctypes.byref(size)) == capi.OK
        assert size.value == want, args
    assert lib.b200_w4_packed_bytes(1, 8, 64, 64, 0, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.b200_w4_packed_bytes(1, 8, 60, 64, 0, ctypes.byref(size)) == \
        capi.ERR_INVALID_ARGUMENT
    assert lib.b200_w4_pack(0, FAKE, 0, FAKE, 1, 8, 64, 64, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.b200_w4_pack(FAKE, FAKE, 0, FAKE + 4, 1, 8, 64, 64, None) == capi.ERR_ALIGNMENT


def test_w4_torch_checks():
    q = torch.zeros(8, 32, dtype=torch.uint8)
    s = torch.zeros(8, 1, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        bg.pack_w4(q, s)
    with pytest.raises(RuntimeError, match="like q"):
        bg.pack_w4(q, s[None])
    with pytest.raises(RuntimeError, match="experts, N, K/2"):
        bg.pack_w4(q[0], s)
    with pytest.raises(RuntimeError, match="multiple of group"):
        bg.quantize_w4(torch.zeros(4, 100, dtype=torch.bfloat16), 64)


def test_route_c_abi():
    lib = capi.lib()

    def route(logits=FAKE, tokens=4, experts=8, ld=8, type=capi.FP32, k=2, w=FAKE, ex=FAKE,
              rows=FAKE, src=FAKE, off=FAKE):
        return lib.b200_route(logits, tokens, experts, ld, type, k, 1, w, ex, rows, src, off, None)

    for change, expect in [(dict(tokens=-1), capi.ERR_INVALID_ARGUMENT),
                           (dict(k=9), capi.ERR_INVALID_ARGUMENT),
                           (dict(k=-1), capi.ERR_INVALID_ARGUMENT),
                           (dict(k=33, experts=64, ld=64), capi.ERR_INVALID_ARGUMENT),
                           (dict(type=3), capi.ERR_INVALID_ARGUMENT),
                           (dict(ld=7), capi.ERR_INVALID_ARGUMENT),
                           (dict(logits=0), capi.ERR_INVALID_ARGUMENT),
                           (dict(off=0), capi.ERR_INVALID_ARGUMENT),
                           (dict(w=0), capi.ERR_INVALID_ARGUMENT),
                           (dict(rows=FAKE + 2), capi.ERR_ALIGNMENT),
                           (dict(logits=FAKE + 2), capi.ERR_ALIGNMENT),
                           (dict(experts=1025, ld=1025), capi.ERR_TOO_LARGE),
                           (dict(tokens=INT_MAX, k=2), capi.ERR_TOO_LARGE)]:
        assert route(**change) == expect, change
    assert lib.b200_route_grad(FAKE, 4, 8, 7, 2, 2, 1, FAKE, FAKE, FAKE, FAKE, None) == \
        capi.ERR_INVALID_ARGUMENT
    assert lib.b200_route_grad(FAKE, 0, 8, 8, 2, 2, 1, FAKE, FAKE, FAKE, FAKE, None) == capi.OK


def test_moving_rows_c_abi():
    lib = capi.lib()
    dispatch = [FAKE, FAKE, FAKE, FAKE, 4, 2, 16, 16, 16, capi.BF16, None]
    combine = [FAKE, FAKE, FAKE, FAKE, 4, 2, 16, 16, 16, capi.BF16, None]
    grad = [FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 4, 2, 16, 16, 16, 16, capi.BF16, None]
    for fn, args, at, value, expect in [
            (lib.b200_dispatch, dispatch, 4, -1, capi.ERR_INVALID_ARGUMENT),
            (lib.b200_dispatch, dispatch, 5, 33, capi.ERR_INVALID_ARGUMENT),
            (lib.b200_dispatch, dispatch, 7, 15, capi.ERR_INVALID_ARGUMENT),
            (lib.b200_dispatch, dispatch, 2, 0, capi.ERR_INVALID_ARGUMENT),
            (lib.b200_dispatch, dispatch, 9, 2, capi.ERR_INVALID_ARGUMENT),
            (lib.b200_dispatch, dispatch, 0, FAKE + 1, capi.ERR_ALIGNMENT),
            (lib.b200_dispatch, dispatch, 4, INT_MAX, capi.ERR_TOO_LARGE),
            (lib.b200_dispatch, dispatch, 4, 0, capi.OK),
            (lib.b200_combine, combine, 2, 0, capi.ERR_INVALID_ARGUMENT),
            (lib.b200_combine, combine, 8, 8, capi.ERR_INVALID_ARGUMENT),
            (lib.b200_combine, combine, 1, FAKE + 2, capi.ERR_ALIGNMENT),
            (lib.b200_combine, combine, 6, 0, capi.OK),
            (lib.b200_combine_grad, grad, 2, 0, capi.ERR_INVALID_ARGUMENT),
            (lib.b200_combine_grad, grad, 4, 0, capi.ERR_INVALID_ARGUMENT),
            (lib.b200_combine_grad, grad, 11, 8, capi.ERR_INVALID_ARGUMENT),
            (lib.b200_combine_grad, grad, 7, 0, capi.OK)]:
        changed = list(args)
        changed[at] = value
        assert fn(*changed) == expect, (fn, at, value)


def test_route_torch_checks():
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        bg.route_b200(x, 2)
    i = torch.zeros(4, 2, dtype=torch.int32)
    r = bg.Routing(torch.zeros(4, 2), i, i, i.flatten(), torch.zeros(9, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        bg.dispatch_b200(x.bfloat16(), r)
    with pytest.raises(RuntimeError, match="2-D"):
        bg.combine_b200(x[0].bfloat16(), r)


def test_align_rows_c_abi():
    lib = capi.lib()
    args = [FAKE, 64, 8, FAKE, 2, 8, 7, 8, None]
    for at, value, expect in [(4, -1, capi.ERR_INVALID_ARGUMENT), (5, -1, capi.ERR_INVALID_ARGUMENT),
                              (7, 6, capi.ERR_INVALID_ARGUMENT), (0, 0, capi.ERR_INVALID_ARGUMENT),
                              (2, -1, capi.ERR_INVALID_ARGUMENT), (0, FAKE + 1, capi.ERR_ALIGNMENT),
                              (3, FAKE + 2, capi.ERR_ALIGNMENT), (7, 12, capi.ERR_ALIGNMENT),
                              (4, 0, capi.OK), (5, 0, capi.OK), (6, 0, capi.OK)]:
        changed = list(args)
        changed[at] = value
        assert lib.b200_align_rows(*changed) == expect, (at, value)
