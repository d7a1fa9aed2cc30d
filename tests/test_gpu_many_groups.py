"""M-grouped products over more groups than a warp has lanes, most of them short or empty, in every row layout and kernel
form: the walk over the group sizes takes 32 groups at a time."""

import pytest
import torch

from gated_ffn_ref import HALF_EPS, assert_within, block
from triton_grouped_gemm_b200 import _lib
from triton_grouped_gemm_b200.gemm.BF16.m_grouped_gated_gemm import m_grouped_gated_gemm
from triton_grouped_gemm_b200.gemm.BF16.m_grouped_gemm_masked_TMA import m_grouped_gemm_masked
from triton_grouped_gemm_b200.gemm.BF16.m_grouped_gemm_TMA import _m_grouped_gemm_launch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _sizes(groups, seed, most, share=0.4):
    gen = torch.Generator().manual_seed(seed)
    s = torch.randint(1, most + 1, (groups,), generator=gen)
    return torch.where(torch.rand(groups, generator=gen) < share, s, torch.zeros_like(s))


def _operands(m, groups, n, k, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    a = torch.randn(m, k, generator=gen, device=DEV).bfloat16()
    b = (torch.randn(groups, n, k, generator=gen, device=DEV) * k ** -0.5).bfloat16()
    return a, b


def _reference(a, b):
    """Rows of one group: (value, bound); fp32 sums err by at most 2^-22 of the magnitudes per 16 products."""
    c = a.double() @ b.double().t()
    e = (a.shape[1] / 16 + 2) * 2.0 ** -22 * (a.double().abs() @ b.double().abs().t())
    return c, e + HALF_EPS[torch.bfloat16] * (c.abs() + e) + 2.0 ** -134


def _check(out, a, b, starts, sizes):
    touched = torch.zeros(out.shape[0], dtype=torch.bool, device=DEV)
    for g, (lo, s) in enumerate(zip(starts, sizes)):
        if s:
            assert_within(out[lo:lo + s], _reference(a[lo:lo + s], b[g]), f"group {g}")
            touched[lo:lo + s] = True
    assert torch.all(out[~touched] == 7.0)


@pytest.mark.parametrize("pair", [-1, 0, 1])
@pytest.mark.parametrize("groups,most", [(33, 3), (64, 200), (70, 40), (300, 5), (1000, 2)])
def test_compact_rows(groups, most, pair):
    sizes = _sizes(groups, groups + most, most)
    m = int(sizes.sum()) + 3
    a, b = _operands(m, groups, 136, 72, groups)
    out = torch.full((m, 136), 7.0, device=DEV, dtype=torch.bfloat16)
    lib = _lib.load()
    lib.b200gemm_set_cta_pair(pair)
    try:
        _m_grouped_gemm_launch(a, b, out, sizes.to(DEV), True)
    finally:
        lib.b200gemm_set_cta_pair(-1)
    assert _lib.device_status() == 0
    _check(out, a, b, (sizes.cumsum(0) - sizes).tolist(), sizes.tolist())


@pytest.mark.parametrize("pair", [-1, 1])
@pytest.mark.parametrize("groups,most", [(70, 3), (129, 40)])
def test_gated_rows(groups, most, pair):
    sizes = _sizes(groups, groups, most)
    m = int(sizes.sum()) + 5
    a, b = _operands(m, groups, 2 * 40, 64, groups)
    out = torch.full((m, 40), 7.0, device=DEV, dtype=torch.bfloat16)
    _lib.load().b200gemm_set_cta_pair(pair)
    try:
        m_grouped_gated_gemm(a, b, sizes.to(DEV), out=out)
    finally:
        _lib.load().b200gemm_set_cta_pair(-1)
    assert _lib.device_status() == 0
    n = int(sizes.sum())
    ref = block(a, b, torch.zeros(groups, 64, 40, device=DEV, dtype=torch.bfloat16), sizes.tolist(), "silu")["h"]
    assert_within(out[:n], tuple(t[:n] for t in ref), "h")
    assert torch.all(out[n:] == 7.0)


@pytest.mark.parametrize("expected", [8, 130])
def test_masked_rows(expected):
    groups = 75
    valid = _sizes(groups, 5, expected + 4)                     # some ask for more than their slot holds
    a, b = _operands(groups * expected, groups, 72, 64, 6)
    out = torch.full((groups * expected, 72), 7.0, device=DEV, dtype=torch.bfloat16)
    m_grouped_gemm_masked(a, b, out, valid.to(DEV), expected)
    assert _lib.device_status() == 0
    _check(out, a, b, [g * expected for g in range(groups)], valid.clamp(max=expected).tolist())


def test_padded_rows():
    groups = 40
    sizes = _sizes(groups, 9, 150)
    padded = (sizes + 127) // 128 * 128
    m = int(padded.sum())
    a, b = _operands(m, groups, 72, 64, 10)
    out = torch.full((m, 72), 7.0, device=DEV, dtype=torch.bfloat16)
    dev = sizes.to(DEV)
    rc = _lib.load().b200gemm_m_grouped_padded(a.data_ptr(), b.data_ptr(), out.data_ptr(), dev.data_ptr(), 1, groups, m, 72, 64, 1,
                                               0, -1, torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "b200gemm_m_grouped_padded")
    assert _lib.device_status() == 0
    _check(out, a, b, (padded.cumsum(0) - padded).tolist(), sizes.tolist())


@pytest.mark.parametrize("bad", [2 ** 31 - 1, 2 ** 62])
def test_sizes_past_the_rows(bad):
    """An absurd size in the second 32 groups: what lies before it is computed, it takes what is left, the rest nothing."""
    groups = 100
    sizes = _sizes(groups, 11, 30, share=1.0)
    m = int(sizes[:61].sum())
    a, b = _operands(m, groups, 72, 64, 12)
    want = sizes.clone()
    want[60:] = 0
    want[60] = m - int(sizes[:60].sum())
    sizes[60] = bad
    sizes[3] = -4
    a3 = int(want[3])
    want[3] = 0
    want[60] += a3
    out = torch.full((m, 72), 7.0, device=DEV, dtype=torch.bfloat16)
    _m_grouped_gemm_launch(a, b, out, sizes.to(DEV), True)
    assert _lib.device_status() == 0x10
    _check(out, a, b, (want.cumsum(0) - want).tolist(), want.tolist())
