"""A caller that works in a driver context of its own keeps it: calls run there
and leave it current.  In a process of its own, without torch."""
import subprocess
import sys
from pathlib import Path

import pytest

PROGRAM = """
import ctypes, sys
sys.path.insert(0, {root!r})
from blackwell_gemm_b200 import capi
cuda = ctypes.CDLL("libcuda.so.1")
P = ctypes.c_void_p
def ok(r): assert r == 0, r
ok(cuda.cuInit(0))
own, seen = P(), P()
ok(cuda.cuCtxCreate_v2(ctypes.byref(own), 0, 0))
def current():
    ok(cuda.cuCtxGetCurrent(ctypes.byref(seen)))
    return seen.value
assert capi.device_status(True) == 0
assert current() == own.value, "the caller's context was replaced"
assert "torch" not in sys.modules
print("kept")
n = 256
words = (ctypes.c_uint16 * (n * n))(*([0x3F80] * (n * n)))   # ones in bf16
ptr = []
for _ in range(3):
    p = P()
    ok(cuda.cuMemAlloc_v2(ctypes.byref(p), ctypes.c_size_t(2 * n * n)))
    ok(cuda.cuMemcpyHtoD_v2(p, words, ctypes.c_size_t(2 * n * n)))
    ptr.append(p.value)
assert capi.gemm_bf16(*ptr, n, n, n, n, n, n, 0) == capi.OK
ok(cuda.cuCtxSynchronize())
assert current() == own.value
ok(cuda.cuMemcpyDtoH_v2(words, P(ptr[2]), ctypes.c_size_t(2 * n * n)))
assert set(words) == {{0x4380}}, sorted(set(words))[:4]      # 256 in bf16
assert capi.device_status(True) == 0
print("computed")
"""


@pytest.mark.gpu
def test_a_context_of_the_callers_own_is_kept():
    root = str(Path(__file__).resolve().parents[1])
    got = subprocess.run([sys.executable, "-c", PROGRAM.format(root=root)], capture_output=True,
                         text=True, timeout=100)
    assert got.returncode == 0, got.stderr[-2000:]
    assert got.stdout.split() == ["kept", "computed"]
