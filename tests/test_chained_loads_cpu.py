"""Kernels that come up while their predecessor runs (launch_chained) must not read through the path for memory that is
read-only as long as the kernel lives: no __ldg, no ld.global.nc, no const __restrict__ pointer in their sources."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "triton_grouped_gemm_b200" / "csrc"
CHAINED = sorted(p.name for p in CSRC.glob("*.cu") if "chain_wait();" in p.read_text())


def _code(text):
    return re.sub(r"//[^\n]*", "", text)


def test_the_chained_sources_are_known():
    assert CHAINED == ["gemm_bf16.cu", "gemm_bf16_k.cu", "gemm_gated.cu", "gemm_k_pair.cu", "gemm_pair.cu", "moe_rows.cu", "w4.cu"]
    launched = {p.name for p in CSRC.glob("*.cu") if "launch_chained" in p.read_text()}
    assert launched <= set(CHAINED)


@pytest.mark.parametrize("name", CHAINED + ["gemm_tile.cuh"])
def test_no_read_only_loads(name):
    code = _code((CSRC / name).read_text())
    if name == "w4.cu":   # the quantiser is launched ordinarily
        code = code[:code.index("w4_quant_kernel")]
    assert "__ldg" not in code and ".nc" not in code
    assert not re.search(r"const\s+\w[\w ]*\*\s*__restrict__", code)


def test_the_walk_over_the_groups():
    code = _code((CSRC / "common.cuh").read_text())
    walker = code[code.index("struct WarpGroupWalker"):]
    assert "__ldg" not in walker and ".nc" not in walker and "__restrict__" not in walker
