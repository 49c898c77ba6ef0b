"""Kernels that begin before the one ahead of them has ended (they call grid_wait) read its
results, so they may not read through the non-coherent path: ld.global.nc is for memory that
nobody writes while the kernel lives, and its life begins before the wait.  A `const T*
__restrict__` parameter lets the compiler take that path by itself."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).parent.parent / "blackwell_gemm_b200" / "csrc"
FILES = [p for p in sorted(CSRC.glob("*.cuh")) if "grid_wait()" in p.read_text()]
# (and what kernels of those files call)
FILES += [CSRC / "ffn_act.cuh", CSRC / "ffn_epilogue.cuh", CSRC / "moe_groups.cuh"]


def code(path):
    text = re.sub(r"/\*.*?\*/", "", path.read_text(), flags=re.S)
    return re.sub(r"//[^\n]*", "", text)


def test_files():
    assert {"ffn_grad.cuh", "grad_norm.cuh", "moe_operands.cuh", "moe_route.cuh",
            "moe_w4.cuh"} <= {p.name for p in FILES}


@pytest.mark.parametrize("path", FILES, ids=lambda p: p.name)
def test_no_non_coherent_loads(path):
    text = code(path)
    assert not re.findall(r"__ldg\s*\(|ld\.global(?:\.\w+)*\.nc", text)
    for m in re.finditer(r"__global__", text):
        head = text[m.start():text.index("{", m.start())]
        assert not re.findall(r"const\s+\w[\w ]*\*\s*(?:const\s+)?__restrict__", head), head
