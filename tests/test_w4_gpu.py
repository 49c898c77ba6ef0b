"""Products with 4-bit weights against the definition in 64 bits.

Tolerance: the output is rounded once (u = 2^-8 bf16, 2^-11 fp16 relative);
before that, fp32 sums of exact products q x, each group's sum times its
scale.  With no assumption on the order of adding or on how the tensor core
rounds (2^-23 an addition), K + 2 roundings of at most sum |x w| each."""
import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi

pytestmark = pytest.mark.gpu

DT = {"bf16": (torch.bfloat16, 2.0 ** -8), "fp16": (torch.float16, 2.0 ** -11)}


@pytest.fixture(autouse=True)
def _clean():
    capi.device_status(True)
    yield
    assert capi.device_status(True) == 0


def weights(e, n, k, group, zeros, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 256, (e, n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = ((torch.rand(e, n, k // group, generator=g, device="cuda") + 0.5) * 0.2 * k ** -0.5).to(dt)
    s[..., ::3] *= -1
    z = None
    if zeros:
        z = torch.randint(0, 16, (e, n, k // group), generator=g, device="cuda", dtype=torch.uint8)
    wide = torch.empty(e, n, k, dtype=torch.float64, device="cuda")
    wide[..., 0::2], wide[..., 1::2] = (q & 15).double(), (q >> 4).double()
    shift = 8.0 if z is None else z.double().repeat_interleave(group, -1)
    return q, s, z, (wide - shift) * s.double().repeat_interleave(group, -1)


def close(got, x, w, u, half=False):
    want, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    bound = 1.0001 * u * want.abs() + 2.0 ** -23 * (x.shape[1] + 2) * size
    if half:
        bound = bound + 2.0 ** -25     # half the smallest fp16 step
    off = (got.double() - want).abs() - bound
    assert bool((off <= 0).all()), float(off.max())


def rows_of(m, k, dt, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(m, k, generator=g, device="cuda").to(dt)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 3, 16, 17, 65])
def test_rows_groups_types(m, group, zeros, dtype):
    dt, u = DT[dtype]
    n, k = 300, 640
    q, s, z, w = weights(1, n, k, group, zeros, dt, seed=m)
    packed = bg.pack_w4(q[0], s[0], None if z is None else z[0])
    x = rows_of(m, k, dt)
    y = bg.matmul_b200_w4(x, packed)
    assert y.shape == (m, n) and y.dtype == dt and y.is_contiguous()
    close(y, x, w[0], u, dtype == "fp16")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [66, 128, 129, 145, 200, 256, 257, 700])
def test_many_rows(m, group, dtype):
    dt, u = DT[dtype]
    n, k = 392, 1120 if group == 32 else 1152
    q, s, z, w = weights(1, n, k, group, m % 2 == 1, dt, seed=m)
    packed = bg.pack_w4(q[0], s[0], None if z is None else z[0])
    x = rows_of(m, k, dt)
    close(bg.matmul_b200_w4(x, packed), x, w[0], u, dtype == "fp16")


@pytest.mark.parametrize("n,k", [(128, 32), (130, 352), (2048, 4096), (5000, 1024)])
def test_many_rows_sizes(n, k):
    # whole and divided contractions, weights past one record and short of one
    q, s, z, w = weights(1, n, k, 32, True, torch.bfloat16, seed=n)
    packed = bg.pack_w4(q[0], s[0], z[0])
    x = rows_of(410, k, torch.bfloat16)
    y = bg.matmul_b200_w4(x, packed)
    close(y, x, w[0], 2.0 ** -8)
    assert torch.equal(y, bg.matmul_b200_w4(x, packed))


@pytest.mark.parametrize("group", [32, 128])
def test_many_rows_of_a_bank(group):
    # experts with none, one, a half, one and a bit and several tiles of rows
    offsets = [3, 3, 4, 132, 393, 393, 1100]
    q, s, z, w = weights(6, 264, 512, group, group == 32, torch.bfloat16)
    x = rows_of(1111, 512, torch.bfloat16)
    x[:3], x[1100:] = float("nan"), float("inf")
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    y = bg.matmul_b200_w4(x, bg.pack_w4(q, s, z), off)
    for e in range(6):
        a, b = offsets[e], offsets[e + 1]
        close(y[a:b], x[a:b], w[e], 2.0 ** -8)
    assert not y[:3].any() and not y[1100:].any()


@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (7, 64, 64), (128, 128, 128), (129, 96, 32),
                                       (1000, 160, 32), (24, 1088, 64), (130, 4096, 128),
                                       (4097, 2048, 128), (512, 14336, 128)])
def test_sizes(n, k, group):
    q, s, z, w = weights(1, n, k, group, True, torch.bfloat16, seed=n)
    packed = bg.pack_w4(q[0], s[0], z[0])
    for m in (1, 40):
        x = rows_of(m, k, torch.bfloat16)
        close(bg.matmul_b200_w4(x, packed), x, w[0], 2.0 ** -8)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("offsets,rows", [([0, 0, 1, 1, 2], 2), ([0, 5, 5, 22, 150], 150),
                                          ([2, 9, 40, 40, 41], 50), ([3, 3, 3, 3, 3], 5)])
def test_bank(offsets, rows, group):
    n, k = 264, 512
    q, s, z, w = weights(4, n, k, group, group == 64, torch.bfloat16)
    packed = bg.pack_w4(q, s, z)
    x = rows_of(rows, k, torch.bfloat16)
    x[:offsets[0]], x[offsets[-1]:] = float("nan"), float("inf")
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    y = bg.matmul_b200_w4(x, packed, off)
    owned = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for e in range(4):
        a, b = offsets[e], offsets[e + 1]
        owned[a:b] = True
        close(y[a:b], x[a:b], w[e], 2.0 ** -8)
    assert not y[~owned].any()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("experts,m", [(1, 2), (1, 20), (1, 50), (1, 140), (1, 300), (2, 100),
                                       (2, 700)])
def test_infinities_and_nan_in_tokens(experts, m, group, dtype):
    # one inf, -inf or NaN in a row: inf with the weight's sign, NaN where it is 0
    dt, _ = DT[dtype]
    n, k = 136, 256
    q, s, z, w = weights(experts, n, k, group, True, dt, seed=m)
    x = rows_of(m, k, dt)
    odd = torch.arange(0, m, 3, device="cuda")
    x[odd, (7 * odd) % k] = float("inf")
    x[odd[1::3], (7 * odd[1::3]) % k] = float("-inf")
    x[odd[2::3], (7 * odd[2::3]) % k] = float("nan")
    off = torch.tensor([0, m // 2, m], dtype=torch.int32, device="cuda")
    if experts == 1:
        y, want = bg.matmul_b200_w4(x, bg.pack_w4(q[0], s[0], z[0])), x.double() @ w[0].T
    else:
        y = bg.matmul_b200_w4(x, bg.pack_w4(q, s, z), off)
        want = torch.cat([x[:m // 2].double() @ w[0].T, x[m // 2:].double() @ w[1].T])
    assert torch.equal(y.isnan(), want.isnan())
    assert torch.equal(y.isposinf(), want.isposinf())
    assert torch.equal(y.isneginf(), want.isneginf())


@pytest.mark.parametrize("group", [32, 64])
def test_every_scale_keeps_its_bits(group):
    # weights m 2^e (q - z) for all 128 significands, in units fp32 sums hold:
    # tokens of one 1 each return the weights themselves
    n, k, m = 128, 512, 512
    s = (1 + torch.arange(n, device="cuda") / 128).bfloat16().repeat_interleave(k // group).view(n, -1)
    q = torch.arange(n * k // 2, device="cuda").mul(73).remainder(256).to(torch.uint8).view(n, -1)
    z = torch.arange(n * k // group, device="cuda").mul(5).remainder(16).to(torch.uint8).view(n, -1)
    wide = torch.stack((q & 15, q >> 4), -1).view(n, k).double()
    w = (wide - z.double().repeat_interleave(group, 1)) * s.double().repeat_interleave(group, 1)
    x = torch.eye(m, device="cuda").bfloat16()
    y = bg.matmul_b200_w4(torch.cat([x, x]), bg.pack_w4(torch.stack([q, q]), torch.stack([s, s]),
                                                        torch.stack([z, z])),
                          torch.tensor([0, m, 2 * m], dtype=torch.int32, device="cuda"))
    assert torch.equal(y[:m], w.T.bfloat16()) and torch.equal(y[m:], w.T.bfloat16())


def test_every_nibble_and_exact_bits():
    # weights, rows and scales whose products and sums fp32 holds exactly
    n, k = 256, 256
    q = torch.arange(n * k // 2, device="cuda").mul(37).remainder(256).to(torch.uint8).view(n, -1)
    s = torch.full((n, k // 64), 0.25, dtype=torch.bfloat16, device="cuda")
    z = torch.arange(n * k // 64, device="cuda").remainder(16).to(torch.uint8).view(n, -1)
    x = torch.randint(-2, 3, (9, k), device="cuda").bfloat16()
    w = torch.stack((q & 15, q >> 4), -1).view(n, k).double()
    w = (w - z.double().repeat_interleave(64, 1)) * 0.25
    assert torch.equal(bg.matmul_b200_w4(x, bg.pack_w4(q, s, z)), (x.double() @ w.T).bfloat16())


def test_strided_rows_and_repeatable_bits():
    n, k = 2048, 4096
    q, s, _, w = weights(1, n, k, 128, False, torch.float16)
    packed = bg.pack_w4(q[0], s[0])
    x = rows_of(11, k, torch.float16)
    wide = torch.zeros(11, k + 16, dtype=torch.float16, device="cuda")
    wide[:, 8:8 + k] = x
    odd = torch.zeros(11, k + 3, dtype=torch.float16, device="cuda")
    odd[:, 1:1 + k] = x
    first = bg.matmul_b200_w4(x, packed)
    close(first, x, w[0], 2.0 ** -11, True)
    for v in (wide[:, 8:8 + k], odd[:, 1:1 + k], x.t().contiguous().t()):
        assert torch.equal(first, bg.matmul_b200_w4(v, packed))
    for _ in range(20):
        assert torch.equal(first, bg.matmul_b200_w4(x, packed))


@pytest.mark.parametrize("m", [5, 25, 60, 150, 400])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_scales_over_the_range(m, group):
    # a power of two in the scales is one in the answer, bit by bit
    q, s, z, _ = weights(2, 136, 256, group, True, torch.bfloat16)
    off = torch.tensor([0, m // 3, m], dtype=torch.int32, device="cuda")
    x = rows_of(m, 256, torch.bfloat16)
    y = bg.matmul_b200_w4(x, bg.pack_w4(q, s, z), off)
    for p in (-80, 80):
        scaled = bg.matmul_b200_w4(x, bg.pack_w4(q, (s.double() * 2.0 ** p).bfloat16(), z), off)
        assert torch.equal(scaled.double(), y.double() * 2.0 ** p)


@pytest.mark.parametrize("group,dtype", [(32, "bf16"), (32, "fp16"), (128, "bf16")])
def test_many_rows_on_other_streams_and_in_graphs(group, dtype):
    dt, u = DT[dtype]
    n, k, m = 640, 2048, 300
    q, s, _, w = weights(1, n, k, group, False, dt)
    packed = bg.pack_w4(q[0], s[0])
    odd = torch.zeros(m, k + 8, dtype=dt, device="cuda")
    odd[:, 8:] = rows_of(m, k, dt)
    x = odd[:, 8:]
    first = bg.matmul_b200_w4(x, packed)
    close(first, x, w[0], u, dtype == "fp16")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = bg.matmul_b200_w4(x, packed)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = bg.matmul_b200_w4(x, packed)
    for _ in range(2):
        y.zero_()
        graph.replay()
        assert torch.equal(first, y)


def test_infinities_follow_the_product():
    n, k = 128, 256
    q, s, _, w = weights(1, n, k, 128, False, torch.bfloat16)
    q[:] = 0x99                                   # every weight is +scale
    s = s.abs()
    x = rows_of(3, k, torch.bfloat16)
    x[1, 7] = float("inf")
    x[2, 200] = float("nan")
    y = bg.matmul_b200_w4(x, bg.pack_w4(q[0], s[0]))
    assert bool(y[0].isfinite().all()) and bool((y[1] == float("inf")).all())
    assert bool(y[2].isnan().all())


def test_quantize_roundtrip():
    w = rows_of(96, 256, torch.bfloat16, seed=5)
    for group in (32, 64, 128):
        q, s = bg.quantize_w4(w, group)
        back = torch.stack((q & 15, q >> 4), -1).view(96, 256).float() - 8
        back = back * s.float().repeat_interleave(group, 1)
        step = s.float().repeat_interleave(group, 1)
        # half a step, and the scale's own rounding (2^-8 of at most 7 steps)
        assert bool(((back - w.float()).abs() <= step * (0.5 + 8 * 2.0 ** -8)).all())
    bank, s = bg.quantize_w4(w.view(2, 48, 256), 64)
    assert bank.shape == (2, 48, 128) and s.shape == (2, 48, 4)


def test_empty_and_refused():
    q, s, z, _ = weights(2, 16, 64, 32, True, torch.bfloat16)
    packed = bg.pack_w4(q[0], s[0])
    assert bg.matmul_b200_w4(rows_of(0, 64, torch.bfloat16), packed).shape == (0, 16)
    x = rows_of(2, 64, torch.bfloat16)
    with pytest.raises(RuntimeError, match="same dtype"):
        bg.matmul_b200_w4(x.half(), packed)
    with pytest.raises(RuntimeError, match="inner dimensions"):
        bg.matmul_b200_w4(x[:, :32], packed)
    with pytest.raises(RuntimeError, match="needs offsets"):
        bg.matmul_b200_w4(x, bg.pack_w4(q, s, z))
    with pytest.raises(RuntimeError, match="no gradient"):
        bg.matmul_b200_w4(x.clone().requires_grad_(True), packed)
    with pytest.raises(RuntimeError, match="offsets must have"):
        bg.matmul_b200_w4(x, bg.pack_w4(q, s, z), torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="32, 64 or 128"):
        bg.pack_w4(q[0], s[0, :, :1].repeat(1, 4))
    with pytest.raises(RuntimeError, match="whole number of groups"):
        bg.pack_w4(q[0], s[0, :, :1].repeat(1, 3))
    with pytest.raises(RuntimeError, match="uint8"):
        bg.pack_w4(q[0].int(), s[0])
    with pytest.raises(RuntimeError, match="bfloat16 or float16"):
        bg.pack_w4(q[0], s[0].float())
    with pytest.raises(RuntimeError, match="zeros"):
        bg.pack_w4(q[0], s[0], z[0].int())


def test_graph_capture():
    q, s, _, _ = weights(1, 4096, 2048, 128, False, torch.bfloat16)
    packed = bg.pack_w4(q[0], s[0])
    x = rows_of(5, 2048, torch.bfloat16)
    bg.matmul_b200_w4(x, packed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = bg.matmul_b200_w4(x, packed)
    for scale in (1.0, 0.5):
        x.mul_(scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, bg.matmul_b200_w4(x, packed))
