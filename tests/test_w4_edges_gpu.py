"""4-bit products where the kernels' rings, scales and arguments meet their ends.

Tolerances are those of test_w4_gpu.py."""
import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi
from test_w4_gpu import DT, close, rows_of, weights

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean():
    capi.device_status(True)
    yield
    assert capi.device_status(True) == 0


@pytest.mark.parametrize("dtype,k,group", [
    ("fp16", 32, 32), ("fp16", 64, 32), ("fp16", 64, 64), ("fp16", 96, 32), ("fp16", 128, 32),
    ("fp16", 128, 64), ("fp16", 128, 128), ("bf16", 128, 128), ("bf16", 384, 128),
    ("bf16", 96, 32), ("bf16", 128, 64)])
def test_short_contractions_through_many_tiles(dtype, k, group):
    # one or three records to a tile, several laps of every ring in each CTA
    dt, u = DT[dtype]
    experts, n = 64, 5504
    q, s, z, w = weights(experts, n, k, group, group != 64, dt, seed=k)
    counts = [33 + (7 * e) % 32 for e in range(experts)]
    offsets = [sum(counts[:e]) for e in range(experts + 1)]
    x = rows_of(offsets[-1], k, dt)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    packed = bg.pack_w4(q, s, z)
    y = bg.matmul_b200_w4(x, packed, off)
    for e in range(experts):
        a, b = offsets[e], offsets[e + 1]
        close(y[a:b], x[a:b], w[e], u, dtype == "fp16")
    for _ in range(3):
        assert torch.equal(y, bg.matmul_b200_w4(x, packed, off))


def test_weights_that_do_not_hold_what_they_say():
    q, s, z, _ = weights(2, 264, 512, 64, True, torch.bfloat16)
    good = bg.pack_w4(q, s, z)
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    x = rows_of(4, 512, torch.bfloat16)
    bg.matmul_b200_w4(x, good, off)
    for change, match in [
            (dict(N=512), "contiguous bytes"), (dict(K=1024), "inner dimensions"),
            (dict(zeros=False), "contiguous bytes"), (dict(experts=1, bank=False), "contiguous"),
            (dict(group=32), "contiguous bytes"), (dict(group=48), "status 1"),
            (dict(group=0), "status 1"), (dict(N=264 + 2 ** 32), "2\\^31"),
            (dict(N=-1), "negative"), (dict(experts=3), "contiguous bytes"),
            (dict(experts=2 ** 32 + 2), "1024 experts"),
            (dict(data=good.data[:-1]), "contiguous bytes"),
            (dict(data=good.data.view(torch.int16)), "contiguous bytes"),
            (dict(data=good.data.repeat_interleave(2)[::2]), "contiguous bytes")]:
        bad = good._replace(**change)
        experts = min(bad.experts, 3)
        ends = None if bad.experts == 1 else torch.arange(experts + 1, dtype=torch.int32,
                                                          device="cuda")
        with pytest.raises(RuntimeError, match=match):
            bg.matmul_b200_w4(x, bad, ends)
    # a copy of it, as a checkpoint gives back, is as good
    again = bg.W4Weight(*[t.clone() if isinstance(t, torch.Tensor) else t for t in good])
    assert torch.equal(bg.matmul_b200_w4(x, again, off), bg.matmul_b200_w4(x, good, off))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("experts,m", [(1, 1), (1, 12), (1, 30), (1, 33), (1, 64), (1, 100), (1, 300),
                                       (2, 90), (2, 700)])
def test_infinite_and_nan_scales(experts, m, group, dtype):
    # an infinite scale makes infinite weights, in kernels for few rows and for many
    dt, u = DT[dtype]
    n, k = 136, 256
    q, s, z, w = weights(experts, n, k, group, True, dt, seed=m)
    nibbles = torch.stack((q & 15, q >> 4), -1).reshape(experts, n, k)
    for row, low in ((3, False), (40, True), (77, False), (135, True)):
        # every weight of this row's first group above its zero point, or below
        nibbles[:, row, :group] = nibbles[:, row, :group] % 7 + (0 if low else 9)
        z[:, row, 0] = 8
    q = (nibbles[..., 0::2] | nibbles[..., 1::2] << 4).contiguous()
    w = (nibbles.double() - z.double().repeat_interleave(group, -1)) * \
        s.double().repeat_interleave(group, -1)
    inf = float("inf")
    for row, scale in ((3, inf), (40, inf), (77, -inf), (135, float("nan"))):
        s[:, row, 0] = scale
    x = rows_of(m, k, dt).abs() + 0.25
    off = torch.tensor([0, m // 2, m], dtype=torch.int32, device="cuda")
    if experts == 1:
        y = bg.matmul_b200_w4(x, bg.pack_w4(q[0], s[0], z[0]))
    else:
        y = bg.matmul_b200_w4(x, bg.pack_w4(q, s, z), off)
    assert bool((y[:, 3] == inf).all()) and bool((y[:, 40] == -inf).all())
    assert bool((y[:, 77] == -inf).all()) and bool(y[:, 135].isnan().all())
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[[3, 40, 77, 135]] = False
    for e in range(experts):
        a, b = (0, m) if experts == 1 else (off[e].item(), off[e + 1].item())
        close(y[a:b, rest], x[a:b], w[e][rest], u, dtype == "fp16")


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [8, 32, 64, 512])
@pytest.mark.parametrize("power", [-120, -110, 119])
def test_small_and_large_scales_keep_their_bits(power, m, group):
    # tokens of one 1 each return the weights themselves
    n, k = 128, 512
    s = (1 + torch.arange(n, device="cuda") / 128).double() * 2.0 ** power
    s = s.bfloat16().repeat_interleave(k // group).view(n, -1)
    q = torch.arange(n * k // 2, device="cuda").mul(73).remainder(256).to(torch.uint8).view(n, -1)
    z = torch.arange(n * k // group, device="cuda").mul(5).remainder(16).to(torch.uint8).view(n, -1)
    wide = torch.stack((q & 15, q >> 4), -1).view(n, k).double()
    w = (wide - z.double().repeat_interleave(group, 1)) * s.double().repeat_interleave(group, 1)
    x = torch.eye(k, device="cuda").bfloat16()[:m]
    assert torch.equal(bg.matmul_b200_w4(x, bg.pack_w4(q, s, z)), w.T[:m].bfloat16())


def test_zero_points_above_15_are_not_taken_silently():
    q, s, z, w = weights(2, 130, 192, 64, True, torch.bfloat16)
    x = rows_of(8, 192, torch.bfloat16)
    off = torch.tensor([0, 4, 8], dtype=torch.int32, device="cuda")
    z[0, 0, 0] = 15
    bg.pack_w4(q, s, z)
    bad = z.clone()
    bad[1, 129, 2] = 16
    with pytest.raises(RuntimeError, match="0 .. 15"):
        bg.pack_w4(q, s, bad)
    with pytest.raises(RuntimeError, match="0 .. 15"):
        bg.pack_w4(q[1], s[1], bad[1])
    # through the C ABI, and in a capture, the device's error word says so
    packed = bg.pack_w4(q, s, z)
    out = torch.empty_like(packed.data)
    stream = torch.cuda.current_stream().cuda_stream

    def pack(zeros, stream):
        return capi.lib().b200_w4_pack(q.data_ptr(), s.data_ptr(), zeros.data_ptr(), out.data_ptr(),
                                       2, 130, 192, 64, stream)
    assert pack(z, stream) == capi.OK and capi.device_status(True) == 0
    assert torch.equal(out, packed.data)
    assert pack(bad, stream) == capi.OK and capi.device_status(True) == 0x100B
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = bg.pack_w4(q, s, z)
        y = bg.matmul_b200_w4(x, again, off)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again.data, packed.data)
    assert torch.equal(y, bg.matmul_b200_w4(x, packed, off))
    z.copy_(bad)
    graph.replay()
    torch.cuda.synchronize()
    assert capi.device_status(True) == 0x100B
