"""What the feed-forward block, the 4-bit products and the row movers refuse, on a machine without a GPU: wrong
arguments at the C entry points (an error code and a message before any device work) and in the Python layer."""

import pytest
import torch

from triton_grouped_gemm_b200 import _lib
from triton_grouped_gemm_b200.ep.autograd import combine_rows, permute_rows
from triton_grouped_gemm_b200.gemm.autograd import grouped_gated_ffn
from triton_grouped_gemm_b200.gemm.BF16.m_grouped_gated_gemm import m_grouped_gated_gemm
from triton_grouped_gemm_b200.gemm.W4.m_grouped_gemm_w4 import m_grouped_gemm_w4, m_grouped_gemm_w4_gated
from triton_grouped_gemm_b200.quant.per_group_cast import per_group_cast_to_w4

P = 16   # a pointer that passes the alignment checks and is never followed


def _refused(rc, text):
    assert rc < 0 and text in _lib.last_error(), (rc, _lib.last_error())


def _gated(a=P, w=P, h=P, saved=None, exps=None, sizes=P, groups=2, rows=4, stride=0, inter=16, k=16, act=0, dtype=0, tail=None,
           tail_cols=0):
    return _lib.load().b200gemm_m_grouped_gated(a, w, h, saved, exps, sizes, 0, groups, rows, stride, inter, k, act, dtype, tail,
                                                tail_cols, -1, None)


def _gated_grad(dy=P, w=P, saved=P, exps=P, dgu=P, sizes=P, groups=2, rows=4, inter=16, k=16, act=0, dtype=0, tail=None, cols=0):
    return _lib.load().b200gemm_m_grouped_gated_grad(dy, w, saved, exps, dgu, sizes, 0, groups, rows, inter, k, act, dtype, tail,
                                                     cols, -1, None)


@pytest.mark.parametrize("call", [_gated, _gated_grad])
def test_gated_entry_points(call):
    _refused(call(dtype=2), "dtype")
    _refused(call(act=2), "activation")
    _refused(call(act=-1), "activation")
    _refused(call(rows=-1), "negative")
    _refused(call(k=0), "k must be positive")
    _refused(call(k=12), "16-byte alignment")
    _refused(call(inter=12), "16-byte alignment")
    _refused(call(w=None), "null")
    _refused(call(w=24), "aligned")
    _refused(call(sizes=None), "null")
    _refused(call(rows=1 << 31), "int32")
    assert call(rows=0, w=None) == 0 and call(inter=0, w=None) == 0 and call(groups=0, w=None) == 0


def test_gated_pairs_of_arguments():
    _refused(_gated(saved=P), "null")                 # the codes without their exponents
    _refused(_gated(exps=P), "null")
    _refused(_gated(saved=8, exps=P), "aligned")
    _refused(_gated(tail=P, tail_cols=12), "tail_cols")
    _refused(_gated(stride=-1), "masked_stride")
    _refused(_gated_grad(exps=None), "null")
    _refused(_gated_grad(dgu=4), "aligned")
    lib = _lib.load()
    assert lib.b200gemm_gated_exponent_bytes(10, 8) == 2 * 10 * 8
    assert lib.b200gemm_gated_exponent_bytes(10, 264) == 2 * 10 * 16
    assert lib.b200gemm_gated_exponent_bytes(-1, 8) == 0


def test_w4_entry_points():
    lib = _lib.load()

    def call(a=P, w=P, s=P, z=None, out=P, sizes=P, groups=2, rows=4, n=16, k=64, gs=32, gated=0, act=0, dtype=0):
        return lib.b200gemm_w4_m_grouped(a, w, s, z, out, sizes, 0, groups, rows, n, k, gs, gated, act, dtype, -1, None)

    _refused(call(dtype=3), "dtype")
    _refused(call(gs=16), "group_size")
    _refused(call(gs=128), "multiple of the group size")
    _refused(call(gated=1, act=5), "activation")
    _refused(call(groups=1025), "1024")
    _refused(call(n=-1), "negative")
    _refused(call(k=0), "k must be positive")
    _refused(call(a=8), "aligned")
    _refused(call(s=3), "aligned")
    _refused(call(w=None), "null")
    _refused(call(rows=1 << 31), "int32")
    assert call(groups=0, w=None) == 0 and call(rows=0, w=None) == 0 and call(n=0, w=None) == 0
    _refused(lib.b200quant_w4_group(P, P, P, None, 4, 100, 32, 0, None), "multiple of the group size")
    _refused(lib.b200quant_w4_group(P, P, P, None, 4, 128, 48, 0, None), "group_size")
    _refused(lib.b200quant_w4_group(None, P, P, None, 4, 128, 64, 0, None), "null")
    assert lib.b200quant_w4_group(None, None, None, None, 0, 128, 64, 0, None) == 0


def test_row_movers():
    lib = _lib.load()
    _refused(lib.b200moe_permute_rows(P, P, P, P, 4, 0, 16, 4, None), "top_k")
    _refused(lib.b200moe_permute_rows(P, P, P, P, 4, 33, 16, 4, None), "top_k")
    _refused(lib.b200moe_permute_rows(P, P, P, P, 4, 2, 12, 8, None), "multiple of 8")
    _refused(lib.b200moe_permute_rows(8, P, P, P, 4, 2, 16, 8, None), "aligned")
    _refused(lib.b200moe_permute_rows(P, None, P, P, 4, 2, 16, 8, None), "null")
    _refused(lib.b200moe_permute_rows(P, P, P, P, -4, 2, 16, 8, None), "negative")
    assert lib.b200moe_permute_rows(None, None, None, None, 0, 2, 16, 0, None) == 0
    _refused(lib.b200moe_combine_rows(P, P, P, P, P, 4, 2, 16, 8, 7, None), "dtype")
    _refused(lib.b200moe_combine_rows(P, P, None, P, P, 4, 2, 16, 8, 0, None), "null")
    assert lib.b200moe_combine_rows(None, None, None, None, None, 0, 2, 16, 0, 0, None) == 0
    _refused(lib.b200moe_combine_rows_grad(P, P, P, P, None, P, P, 4, 2, 16, 8, 0, None), "null")
    _refused(lib.b200moe_combine_rows_grad(P, None, P, P, P, P, P, 4, 2, 16, 8, 0, None), "null")
    _refused(lib.b200moe_combine_rows_grad(P, P, P, P, P, 8, P, 4, 2, 16, 8, 0, None), "aligned")
    assert lib.b200moe_combine_rows_grad(None, None, None, None, None, None, None, 4, 2, 16, 8, 0, None) == 0


def test_python_layer():
    bf = torch.bfloat16
    x, w13, w2 = torch.zeros(4, 16, dtype=bf), torch.zeros(2, 32, 16, dtype=bf), torch.zeros(2, 16, 16, dtype=bf)
    s = torch.tensor([2, 2])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        grouped_gated_ffn(x, w13, w2, s)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        m_grouped_gated_gemm(x, w13, s)
    for bad in (w2[:1], w2[:, :8], w2[:, :, :8]):
        with pytest.raises(AssertionError, match="w2 should have shape"):
            grouped_gated_ffn(x, w13, bad, s)
    with pytest.raises(AssertionError, match="dtype"):
        grouped_gated_ffn(x, w13, w2.half(), s)
    with pytest.raises(AssertionError, match="activation"):
        m_grouped_gated_gemm(x, w13, s, "relu")
    with pytest.raises(AssertionError, match="not supported"):
        m_grouped_gated_gemm(x.float(), w13.float(), s)
    with pytest.raises(AssertionError, match="K of A"):
        m_grouped_gated_gemm(x[:, :8].contiguous(), w13, s)
    with pytest.raises(AssertionError, match="one entry per group"):
        m_grouped_gated_gemm(x, w13, s[:1])
    q, sc = torch.zeros(2, 6, 32, dtype=torch.uint8), torch.zeros(2, 6, 2, dtype=bf)
    a = torch.zeros(4, 64, dtype=bf)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        m_grouped_gemm_w4(a, (q, sc, None), s)
    with pytest.raises(AssertionError, match="K mismatch"):
        m_grouped_gemm_w4(a[:, :32], (q, sc, None), s)
    with pytest.raises(AssertionError, match="scale must have a's dtype"):
        m_grouped_gemm_w4(a, (q, sc.half(), None), s)
    with pytest.raises(AssertionError, match="group_size"):
        m_grouped_gemm_w4(a, (q, torch.zeros(2, 6, 4, dtype=bf), None), s)
    with pytest.raises(AssertionError, match="zero must be"):
        m_grouped_gemm_w4(a, (q, sc, sc), s)
    with pytest.raises(AssertionError, match="gate rows"):
        m_grouped_gemm_w4_gated(a, (q[:, :5].contiguous(), sc[:, :5].contiguous(), None), s)
    with pytest.raises(AssertionError, match="group_size"):
        per_group_cast_to_w4(torch.zeros(4, 96, dtype=bf), 64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        per_group_cast_to_w4(torch.zeros(4, 64, dtype=bf), 64)
    pos = torch.arange(8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        permute_rows(x, pos, pos, 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        combine_rows(torch.zeros(8, 16, dtype=bf), torch.zeros(4, 2), pos, pos)
    with pytest.raises(AssertionError, match="order must have one entry per row"):
        combine_rows(torch.zeros(7, 16, dtype=bf), torch.zeros(4, 2), pos, pos)
