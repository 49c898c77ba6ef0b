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
