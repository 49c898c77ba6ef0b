"""Calls from several host threads at once, each on a stream of its own.

cudaStreamPerThread is one handle that names another stream in every thread;
what the library keeps per stream (arrival counts, flags, tickets) must not be
shared between them.  Inputs are small whole numbers, every sum is exact, so
each result has to equal the single-threaded one bit for bit."""
import ctypes
import threading

import pytest
import torch

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi

pytestmark = pytest.mark.gpu

PER_THREAD = 2  # cudaStreamPerThread


@pytest.fixture(autouse=True)
def _clean():
    yield
    capi.set_dynamic(0)
    capi.set_stream_k(1)
    assert capi.device_status(True) == 0


def whole(*shape, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-2, 3, shape, generator=g, device="cuda").to(dtype)


def in_threads(call, out, want, threads=3, rounds=40):
    """call(stream, out[i]) `rounds` times in each thread; every result against want."""
    torch.cuda.synchronize()
    runtime = ctypes.CDLL("libcudart.so.12")
    start = threading.Barrier(threads)
    status = [[] for _ in range(threads)]

    def work(i):
        start.wait()
        for r in range(rounds):
            status[i].append(call(PER_THREAD, out[i][r]))
        # (the stream goes with its thread: nothing may still run on it)
        status[i].append(runtime.cudaStreamSynchronize(ctypes.c_void_p(PER_THREAD)))

    team = [threading.Thread(target=work, args=(i,)) for i in range(threads)]
    for t in team:
        t.start()
    for t in team:
        t.join()
    torch.cuda.synchronize()
    assert all(s == capi.OK for each in status for s in each)
    for i in range(threads):
        for r in range(rounds):
            assert torch.equal(out[i][r], want), (i, r)


def outputs(*shape, threads=3, rounds=40):
    return torch.zeros(threads, rounds, *shape, dtype=torch.bfloat16, device="cuda")


def test_grouped_product():
    rows, experts, n, k = 12, 4, 640, 4096
    x, w = whole(rows, k), whole(experts, n, k, seed=1)
    off = torch.tensor([0, 3, 6, 9, 12], dtype=torch.int32, device="cuda")
    want = bg.matmul_b200_grouped(x, w.transpose(1, 2), off)

    def call(stream, out):
        return capi.lib().b200_grouped_gemm(x.data_ptr(), w.data_ptr(), out.data_ptr(),
                                            off.data_ptr(), rows, experts, n, k, k, k, n * k, n,
                                            capi.BF16, stream)
    in_threads(call, outputs(rows, n), want)


@pytest.mark.parametrize("rows,group", [(1, 128), (12, 128), (24, 32), (50, 128), (50, 32),
                                        (120, 32), (200, 128)])
def test_4bit_product(rows, group):
    n, k = 640, 4096
    x = whole(rows, k)
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    weight = bg.pack_w4(q, torch.ones(n, k // group, dtype=torch.bfloat16, device="cuda"))
    want = bg.matmul_b200_w4(x, weight)

    def call(stream, out):
        return capi.lib().b200_w4_gemm(x.data_ptr(), weight.data.data_ptr(), out.data_ptr(), None,
                                       rows, 1, n, k, group, 0, k, n, capi.BF16, stream)
    in_threads(call, outputs(rows, n), want)


@pytest.mark.parametrize("dynamic,m,n,k", [(0, 768, 6400, 4096), (0, 16, 4000, 8192),
                                           (1, 2048, 6400, 512)])
def test_matmul(dynamic, m, n, k):
    capi.set_dynamic(dynamic)
    a, b = whole(m, k), whole(n, k, seed=1)
    want = (a.double() @ b.double().T).bfloat16()

    def call(stream, out):
        return capi.gemm_bf16(a.data_ptr(), b.data_ptr(), out.data_ptr(), m, n, k, k, k, n, stream)
    in_threads(call, outputs(m, n, rounds=10), want, rounds=10)


def test_streams_made_and_destroyed():
    # more streams than there are places for, handles coming back among them
    rows, experts, n, k = 4, 2, 640, 4096
    x, w = whole(rows, k), whole(experts, n, k, seed=1)
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    want = bg.matmul_b200_grouped(x, w.transpose(1, 2), off)
    runtime = ctypes.CDLL("libcudart.so.12")
    out = outputs(rows, n, threads=1, rounds=300)[0]
    torch.cuda.synchronize()
    for r in range(300):
        stream = ctypes.c_void_p()
        assert runtime.cudaStreamCreate(ctypes.byref(stream)) == 0
        assert capi.lib().b200_grouped_gemm(x.data_ptr(), w.data_ptr(), out[r].data_ptr(),
                                            off.data_ptr(), rows, experts, n, k, k, k, n * k, n,
                                            capi.BF16, stream) == capi.OK
        assert runtime.cudaStreamDestroy(stream) == 0
    torch.cuda.synchronize()
    assert all(torch.equal(out[r], want) for r in range(300))


@pytest.mark.parametrize("what", ["grouped", "w4", "stream-K", "dealing"])
def test_calls_while_another_thread_captures(what):
    # nothing that a call allocates may end a capture (global mode) elsewhere
    rows, n, k = 4, 640, 4096
    x, w = whole(rows, k), whole(2, n, k, seed=1)
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    weight = bg.pack_w4(*bg.quantize_w4(w[0]))
    a, b = whole(2048, 512), whole(6400, 512, seed=1)
    x16, wide = whole(16, k), whole(1280, k, seed=1)
    side = torch.cuda.Stream()
    stream = side.cuda_stream
    out = {"grouped": (rows, n), "w4": (rows, n), "stream-K": (16, 1280), "dealing": (2048, 6400)}[what]
    out = torch.zeros(*out, dtype=torch.bfloat16, device="cuda")
    lib = capi.lib()
    capi.set_dynamic(1 if what == "dealing" else 0)
    call = {
        "grouped": lambda: lib.b200_grouped_gemm(x.data_ptr(), w.data_ptr(), out.data_ptr(),
                                                 off.data_ptr(), rows, 2, n, k, k, k, n * k, n,
                                                 capi.BF16, stream),
        "w4": lambda: lib.b200_w4_gemm(x.data_ptr(), weight.data.data_ptr(), out.data_ptr(), None,
                                       rows, 1, n, k, 128, 0, k, n, capi.BF16, stream),
        "stream-K": lambda: capi.gemm_bf16(x16.data_ptr(), wide.data_ptr(), out.data_ptr(), 16, 1280,
                                           k, k, k, 1280, stream),
        "dealing": lambda: capi.gemm_bf16(a.data_ptr(), b.data_ptr(), out.data_ptr(), 2048, 6400, 512,
                                          512, 512, 6400, stream),
    }[what]
    want = {"grouped": lambda: bg.matmul_b200_grouped(x, w.transpose(1, 2), off),
            "w4": lambda: bg.matmul_b200_w4(x, weight),
            "stream-K": lambda: (x16.double() @ wide.double().T).bfloat16(),
            "dealing": lambda: (a.double() @ b.double().T).bfloat16()}[what]()
    if what == "stream-K":
        capi.set_skinny_mode(3)
    got = []
    team = threading.Thread(target=lambda: got.extend([call(), call()]))
    static = torch.ones(8, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, capture_error_mode="global"):
            doubled = static * 2
            team.start()
            team.join()
    finally:
        capi.set_skinny_mode(1)
    graph.replay()
    torch.cuda.synchronize()
    assert got == [capi.OK, capi.OK] and bool((doubled == 2).all())
    assert torch.equal(out, want)


@pytest.mark.parametrize("rows,experts", [(12, 4), (50, 1), (300, 1)])
def test_two_streams_at_once(rows, experts):
    # nothing orders the streams: each has counts and slots of its own
    n, k = 640, 4096
    x, w = whole(rows, k), whole(experts, n, k, seed=1)
    off = (torch.arange(experts + 1, device="cuda") * rows // experts).int()
    weight = bg.pack_w4(*bg.quantize_w4(w, 32))
    calls = (lambda: bg.matmul_b200_grouped(x, w.transpose(1, 2), off),
             lambda: bg.matmul_b200_w4(x, weight, off))
    want = [call() for call in calls]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for r in range(60):
        with torch.cuda.stream(streams[r % 3]):
            got.append((r % 2, calls[r % 2]()))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[which]) for which, y in got)
