"""Arguments of the mixture-of-experts operators at the ends of their types."""
import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad,seen", [
    ([0, 5, 2 ** 32 + 8], [0, 5, 12]), ([0, 2 ** 32 + 5, 8], [0, 12, 12]),
    ([-2 ** 32, 5, 12], [0, 5, 12]), ([2 ** 33, 2 ** 33, 2 ** 33], [12, 12, 12]),
    ([-2 ** 63, 2 ** 63 - 1, 12], [0, 12, 12])])
def test_offsets_past_32_bits_are_clamped_and_reported(bad, seen):
    # int64 offsets: clamped to the rows as they are, not what 32 bits keep of them
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(12, 64, generator=g, device="cuda").bfloat16()
    w = torch.randn(2, 64, 40, generator=g, device="cuda").bfloat16()
    q, s = bg.quantize_w4(w.transpose(1, 2).contiguous(), 64)
    weight = bg.pack_w4(q, s)
    bad = torch.tensor(bad, dtype=torch.int64, device="cuda")
    good = torch.tensor(seen, dtype=torch.int64, device="cuda")
    capi.device_status(True)
    for call in (lambda off: bg.matmul_b200_grouped(x, w, off),
                 lambda off: bg.matmul_b200_w4(x, weight, off)):
        want = call(good)
        assert capi.device_status(True) == 0
        assert torch.equal(call(bad), want)
        assert capi.device_status(True) == 0x100A
    strided = torch.stack((good, good), 1)[:, 0]
    assert torch.equal(bg.matmul_b200_grouped(x, w, strided), bg.matmul_b200_grouped(x, w, good))
    assert capi.device_status(True) == 0
