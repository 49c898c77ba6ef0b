"""A refusal whose message holds a number is an exception (formatting one used
to crash the process when two C++ runtimes were linked into it), and a thread
that has not used CUDA yet can call the library."""
import threading

import pytest

import blackwell_gemm_b200 as bg
from blackwell_gemm_b200 import capi


def test_number_in_an_error_message():
    with pytest.raises(RuntimeError, match=r"status 1\)"):
        bg.load().profile_rows(-1, 8, 8)


@pytest.mark.gpu
def test_call_from_a_thread_without_a_context():
    import torch
    a = torch.ones(64, 64, dtype=torch.bfloat16, device="cuda")
    c = torch.empty_like(a)
    torch.cuda.synchronize()
    got = []
    ptrs = (a.data_ptr(), a.data_ptr(), c.data_ptr())
    t = threading.Thread(target=lambda: got.append(
        capi.gemm_bf16(*ptrs, 64, 64, 64, 64, 64, 64, 0)))
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert got == [capi.OK] and bool((c == 64).all())
