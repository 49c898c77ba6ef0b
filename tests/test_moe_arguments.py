"""Arguments of the mixture-of-experts entry points that are refused before any
device is touched."""
from blackwell_gemm_b200 import capi

FAKE = 0x7F0000000000  # never dereferenced: validation fails or returns first


def test_narrow_offsets():
    call = capi.lib().b200_narrow_offsets
    assert call(FAKE, 1, -1, FAKE, None) == capi.ERR_INVALID_ARGUMENT
    assert call(FAKE, -1, 3, FAKE, None) == capi.ERR_INVALID_ARGUMENT
    assert call(None, 1, 3, FAKE, None) == capi.ERR_INVALID_ARGUMENT
    assert call(FAKE, 1, 3, None, None) == capi.ERR_INVALID_ARGUMENT
    assert call(FAKE + 4, 1, 3, FAKE, None) == capi.ERR_ALIGNMENT
    assert call(FAKE, 1, 3, FAKE + 2, None) == capi.ERR_ALIGNMENT
    assert call(FAKE, 1, 1026, FAKE, None) == capi.ERR_TOO_LARGE
    assert call(None, 1, 0, None, None) == capi.OK


def test_route_gradient_alignment():
    call = capi.lib().b200_route_grad
    for type, size in ((capi.FP32, 4), (capi.BF16, 2), (capi.FP16, 2)):
        good = [FAKE, 4, 8, 8, type, 2, 1, FAKE, FAKE, FAKE, FAKE, None]
        for at, by in ((0, size // 2), (7, 2), (8, 2), (9, 2), (10, size // 2)):
            args = list(good)
            args[at] += by
            assert call(*args) == capi.ERR_ALIGNMENT, (type, at)


def test_extents_that_32_bit_indexes_could_pass():
    # a tile, a chunk or a block's step more must not leave 32 bits
    lib, most = capi.lib(), 2 ** 31 - 2 ** 25
    for big in (most + 1, 2 ** 31 - 8):
        ld, far = big // 8 * 8 + 8 if big + 8 < 2 ** 31 else 2 ** 31 - 8, 2 ** 40

        def grouped(rows=8, n=8, k=8, ldn=8, ldk=8):
            return (lib.b200_grouped_gemm(FAKE, FAKE, FAKE, FAKE, rows, 2, n, k, ldk, ldk, far, ldn,
                                          capi.BF16, None),
                    lib.b200_grouped_gemm_da(FAKE, FAKE, FAKE, FAKE, rows, 2, n, k, ldn, ldk, far, ldk,
                                             capi.BF16, None),
                    lib.b200_grouped_gemm_db(FAKE, FAKE, FAKE, FAKE, rows, 2, n, k, ldn, ldk, ldk, far,
                                             capi.BF16, None))
        for change in (dict(rows=big), dict(n=big, ldn=ld)):
            assert grouped(**change) == (capi.ERR_TOO_LARGE,) * 3, change
        if ld >= big:
            assert grouped(k=big, ldk=ld) == (capi.ERR_TOO_LARGE,) * 3
        for rows, n in ((big, 8), (8, big)):
            assert lib.b200_w4_gemm(FAKE, FAKE, FAKE, None, rows, 1, n, 64, 64, 0, 64, max(n, 8),
                                    capi.BF16, None) == capi.ERR_TOO_LARGE
        assert lib.b200_route(FAKE, big, 8, 8, capi.FP32, 1, 1, FAKE, FAKE, FAKE, FAKE, FAKE,
                              None) == capi.ERR_TOO_LARGE
        assert lib.b200_route_grad(FAKE, big, 8, 8, capi.FP32, 1, 1, FAKE, FAKE, FAKE, FAKE,
                                   None) == capi.ERR_TOO_LARGE
        for tokens, width in ((big, 16), (4, big)):
            assert lib.b200_dispatch(FAKE, FAKE, FAKE, FAKE, tokens, 1, width, big, big, capi.BF16,
                                     None) == capi.ERR_TOO_LARGE
            assert lib.b200_combine(FAKE, FAKE, FAKE, FAKE, tokens, 1, width, big, big, capi.BF16,
                                    None) == capi.ERR_TOO_LARGE
            assert lib.b200_combine_grad(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, tokens, 1, width,
                                         big, big, big, capi.BF16, None) == capi.ERR_TOO_LARGE
        assert lib.b200_align_rows(FAKE, 0, 8, FAKE, 1, 8, big, ld if ld >= big else 2 ** 31 - 8,
                                   None) == capi.ERR_TOO_LARGE


def test_quantize_tiny_weights():
    # nearest multiple of the scale, however small that is; zeros stay zero
    import torch
    import blackwell_gemm_b200 as bg
    g = torch.Generator().manual_seed(0)
    for power in (0, -60, -110):
        w = (torch.randn(16, 256, generator=g).double() * 2.0 ** power).bfloat16()
        w[3, :64] = 0
        q, s = bg.quantize_w4(w, 64)
        nibbles = torch.stack((q & 15, q >> 4), -1).view(16, 256).double()
        back = (nibbles - 8) * s.double().repeat_interleave(64, 1)
        # half a step; the largest may stand 7 (1 + 2^-8) steps out
        assert bool(((back - w.double()).abs() <=
                     s.double().repeat_interleave(64, 1) * (0.5 + 2.0 ** -20)).all()), power
        assert not back[3, :64].any()
