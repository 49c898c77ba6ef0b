"""Gated products over banks of 128 to 1024 experts: the last bank whose table fits beside
all stages, the first that takes a stage's place, and the largest.  Most experts have no rows
or a few, one has more than a tile holds, and rows at both ends belong to nobody.

Against products in 64 bits, with the tolerances of test_gated_gpu.py."""
import pytest
import torch

from blackwell_gemm_b200 import capi
from test_gated_gpu import DT, KERNELS, check

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean():
    capi.device_status(True)
    yield
    capi.ffn_set_kernel(0)
    assert capi.device_status(True) == 0


def layout(experts, seed):
    """Offsets with 2 rows before the first expert's, and the rows of the operand: 5 more."""
    r = torch.Generator().manual_seed(seed)
    counts = torch.randint(1, 6, (experts,), generator=r)
    counts[torch.rand(experts, generator=r) < 0.6] = 0
    large = torch.randperm(experts, generator=r)[:3]
    counts[large[0]], counts[large[1]], counts[large[2]] = 300, 70, 17
    ends = [2, *(2 + counts.cumsum(0)).tolist()]
    return ends, ends[-1] + 5


# 72 x 136 as it lies; 33 x 75 through aligned copies, its weights' gradients by plain stores
@pytest.mark.parametrize("n,k", [(72, 136), (33, 75)])
@pytest.mark.parametrize("kernel", ["chosen", "stream", "pair"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("experts", [128, 129, 200, 1024])
def test_banks(experts, dtype, kernel, n, k):
    capi.ffn_set_kernel(KERNELS[kernel])
    offsets, rows = layout(experts, experts)
    check(offsets, rows, n, k, dtype, off_dtype=torch.int64 if dtype == "fp16" else torch.int32)


@pytest.mark.parametrize("kernel", ["stream", "pair"])
def test_wide(kernel):
    """Several tiles of features and columns, and a long contraction, of each expert."""
    capi.ffn_set_kernel(KERNELS[kernel])
    offsets, rows = layout(160, 7)
    check(offsets, rows, 392, 520, "bf16", "gelu")


@pytest.mark.parametrize("kernel", ["stream", "pair"])
def test_last_expert_only(kernel):
    capi.ffn_set_kernel(KERNELS[kernel])
    check([0] * 1024 + [90], 90, 72, 136)
    check([0] + [90] * 1024, 90, 72, 136)
