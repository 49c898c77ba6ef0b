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


@pytest.mark.parametrize("n,k", [(512, 1024), (512, 1021), (509, 1024)])
def test_one_copy_of_an_operand_that_is_not_read_as_it_lies(n, k):
    # a bank that lies as (experts, K, N), rows that lie as (K, rows)
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randn(8, k, n, generator=g, device="cuda").bfloat16()
    x = torch.randn(k, 640, generator=g, device="cuda").bfloat16().t()
    off = torch.arange(9, dtype=torch.int32, device="cuda") * 80
    want = torch.cat([x[80 * e:80 * e + 80].double() @ w[e].double() for e in range(8)])
    bg.matmul_b200_grouped(x, w, off)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y = bg.matmul_b200_grouped(x, w, off)
    extra = torch.cuda.max_memory_allocated() - before
    pad = (k + 7) // 8 * 8
    copies = 8 * n * pad * 2 + 640 * pad * 2
    # (the allocator leaves up to 1 MB of a cached block with an allocation)
    assert extra <= copies + 640 * n * 2 + 3 * 2 ** 20 < copies + 8 * n * k * 2, (extra, copies)
    size = torch.cat([x[80 * e:80 * e + 80].double().abs() @ w[e].double().abs() for e in range(8)])
    bound = 1.0001 * 2.0 ** -8 * want.abs() + 2.0 ** -23 * (k + 2) * size
    assert bool(((y.double() - want).abs() <= bound).all())
