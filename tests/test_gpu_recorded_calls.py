"""Traced calls of the new operators compute on the inputs they are replayed with, and 4-bit products say that they have no
gradient where one is asked for."""

import warnings

import pytest
import torch

from triton_grouped_gemm_b200 import _lib
from triton_grouped_gemm_b200.ep.autograd import combine_rows, permute_rows
from triton_grouped_gemm_b200.gemm.autograd import grouped_gated_ffn
from triton_grouped_gemm_b200.gemm.BF16.m_grouped_gated_gemm import m_grouped_gated_gemm
from triton_grouped_gemm_b200.gemm.W4.m_grouped_gemm_w4 import m_grouped_gemm_w4, m_grouped_gemm_w4_gated
from triton_grouped_gemm_b200.quant.per_group_cast import per_group_cast_to_w4

pytestmark = pytest.mark.gpu


def _operands():
    gen = torch.Generator(device="cuda").manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()  # noqa: E731
    sizes = torch.tensor([5, 0, 9], device="cuda")
    order = torch.randperm(14, generator=gen, device="cuda")
    pos = torch.empty_like(order)
    pos[order] = torch.arange(14, device="cuda")
    return n, sizes, pos, order, n(3, 64, 64), n(3, 64, 32), torch.rand(7, 2, generator=gen, device="cuda")


def test_traces_compute_on_new_inputs():
    n, sizes, pos, order, w13, w2, weight = _operands()
    g13, g2 = per_group_cast_to_w4(w13, 32), per_group_cast_to_w4(w2, 32, symmetric=False)

    def layer(x):
        rows = permute_rows(x, pos, order, 2)
        y = grouped_gated_ffn(rows, w13, w2, sizes)
        h = m_grouped_gated_gemm(rows, w13, sizes)
        return (combine_rows(y, weight, pos, order), m_grouped_gemm_w4(h, g2, sizes),
                m_grouped_gemm_w4(m_grouped_gemm_w4_gated(rows, g13, sizes), g2, sizes))

    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        traced = torch.jit.trace(layer, (n(7, 64),), check_trace=False)
    for _ in range(2):
        x = n(7, 64)
        for a, b in zip(traced(x), layer(x)):
            assert torch.equal(a, b)
    assert _lib.device_status() == 0


def test_four_bit_products_refuse_a_gradient():
    n, sizes, _, _, w13, _, _ = _operands()
    b = per_group_cast_to_w4(w13, 32)
    x = n(14, 64).requires_grad_()
    y = m_grouped_gemm_w4_gated(x, b, sizes)
    with torch.no_grad():
        assert torch.equal(y, m_grouped_gemm_w4_gated(x, b, sizes))
    with pytest.raises(RuntimeError, match="no gradient"):
        y.sum().backward()
    out = torch.empty(14, 32, device="cuda", dtype=torch.bfloat16)
    assert not m_grouped_gemm_w4_gated(x, b, sizes, out=out).requires_grad and torch.equal(out, y)
