"""M-grouped products with 4-bit weights and group scales, for the few rows per expert of a decoding step.

Weights are what ``quant.per_group_cast.per_group_cast_to_w4`` produces:

    b = (w4 [G, N, K/2] uint8, scale [G, N, K/group_size], zero [G, N, K/group_size] uint8 or None)
    C[r, n] = sum_grp scale[g, n, grp] * sum_{k in grp} (q[g, n, k] - zero[g, n, grp]) * a[r, k]

Element 2j of a row is the low half of byte j, element 2j+1 the high half; a ``zero`` is a whole number 0..15 (not
checked: beyond 15 bf16 and fp16 need not agree), ``zero=None`` stands for 8 everywhere;
``scale`` has the type of ``a`` (bf16 or fp16).  The reference has no 4-bit path.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from ... import _lib
from ..BF16.m_grouped_gated_gemm import activation_code

W4Weight = Tuple[Tensor, Tensor, Optional[Tensor]]


class _W4Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, w4, scale, zero, size_per_group, gated, act, num_sms):
        return _launch(a, (w4, scale, zero), size_per_group, gated, act, None, num_sms)

    @staticmethod
    def backward(ctx, dc):
        raise RuntimeError("the 4-bit products have no gradient")


def _product(a: Tensor, b: W4Weight, size_per_group: Tensor, gated: bool, act: int, out: Optional[Tensor],
             num_sms: int) -> Tensor:
    if out is not None:
        _lib.refuse_recorded_out("a 4-bit product", a, b[1])
    elif _lib.recorded("a 4-bit product", a, b[1]):
        return _W4Product.apply(a, *b, size_per_group, gated, act, num_sms)
    return _launch(a, b, size_per_group, gated, act, out, num_sms)


def _launch(a: Tensor, b: W4Weight, size_per_group: Tensor, gated: bool, act: int, out: Optional[Tensor],
            num_sms: int) -> Tensor:
    w4, scale, zero = b
    assert a.dim() == 2, "a must be 2D [M, K]"
    assert w4.dim() == 3 and w4.dtype == torch.uint8, "w4 must be uint8 [num_groups, N, K/2]"
    m, k = a.shape
    g, rows, half = w4.shape
    assert half * 2 == k, f"K mismatch: a has K={k}, w4 has K={half * 2}"
    code = _lib.dtype_code(a.dtype)
    assert scale.dim() == 3 and scale.shape[0] == g and scale.shape[1] == rows and scale.shape[2] > 0, \
        "scale must be [num_groups, N, K/group_size]"
    group_size = k // scale.shape[2]
    assert group_size in (32, 64, 128) and group_size * scale.shape[2] == k, "group_size must be 32, 64 or 128 and divide K"
    assert scale.dtype == a.dtype, "scale must have a's dtype"
    assert a.is_contiguous() and w4.is_contiguous() and scale.is_contiguous()
    if zero is not None:
        assert zero.shape == scale.shape and zero.dtype == torch.uint8 and zero.is_contiguous(), \
            "zero must be uint8 of scale's shape"
        _lib.require_cuda(zero)
        assert zero.get_device() == a.get_device(), "all operands must be on one device"
    assert not gated or rows % 2 == 0, "gated weights hold as many gate rows as up rows"
    n = rows // 2 if gated else rows
    assert size_per_group.numel() == g, "size_per_group must have one entry per group"
    _lib.require_cuda(a, w4, scale, size_per_group)
    assert a.get_device() == w4.get_device() == scale.get_device() == size_per_group.get_device(), \
        "all operands must be on one device"
    if out is None:
        out = a.new_empty(m, n)
    else:
        assert out.shape == (m, n) and out.dtype == a.dtype and out.is_contiguous() and out.device == a.device, \
            "out should be contiguous, of a's type and device and of shape [M, N]"
    sizes, is64 = _lib.sizes_arg(size_per_group)
    device = a.device
    with _lib.on_device(device):
        rc = _lib.load().b200gemm_w4_m_grouped(
            _lib.ptr(a), _lib.ptr(w4), _lib.ptr(scale), _lib.ptr(zero) if zero is not None else None, _lib.ptr(out),
            _lib.ptr(sizes), is64, g, m, n, k, group_size, 1 if gated else 0, act, code, int(num_sms),
            _lib.stream_ptr(device))
    _lib.check(rc, "b200gemm_w4_m_grouped")
    return out


def m_grouped_gemm_w4(a: Tensor, b: W4Weight, size_per_group: Tensor, *, out: Optional[Tensor] = None,
                      num_sms: int = -1) -> Tensor:
    """[M, N] of a [M, K] (compact rows grouped by expert) and the 4-bit weights ``b``.  N needs no alignment, at
    most 1024 groups.  Rows behind ``sum(size_per_group)`` are left as they were in ``out``.  Made for few rows
    per expert; any number is accepted.  No gradient: differentiating through the result raises (``out`` is written outside
    autograd)."""
    return _product(a, b, size_per_group, False, 0, out, num_sms)


def m_grouped_gemm_w4_gated(a: Tensor, b: W4Weight, size_per_group: Tensor, activation: str = "silu", *,
                            out: Optional[Tensor] = None, num_sms: int = -1) -> Tensor:
    """[M, I] ``act(a @ Wg_g.T) * (a @ Wu_g.T)`` with 4-bit weights of 2*I rows per expert (gate rows, then up
    rows) in one kernel; ``activation`` "silu" or "gelu_tanh"."""
    return _product(a, b, size_per_group, True, activation_code(activation), out, num_sms)
