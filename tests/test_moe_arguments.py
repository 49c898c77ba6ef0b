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
