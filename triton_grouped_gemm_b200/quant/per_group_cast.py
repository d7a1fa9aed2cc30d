"""4-bit weight quantiser with group scales along K (the format of ``gemm.W4.m_grouped_gemm_w4``)."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _lib


def per_group_cast_to_w4(w: torch.Tensor, group_size: int = 128, symmetric: bool = True) \
        -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """w [..., K] bf16 / fp16 (finite) -> (uint8 [..., K/2], scales [..., K/group_size] of w's type, zeros uint8
    [..., K/group_size] or None).  ``symmetric``: w ~ (q - 8) * scale with scale = max|w| / 7; otherwise
    w ~ (q - zero) * scale with scale = (max(w, 0) - min(w, 0)) / 15.  group_size 32, 64 or 128, dividing K."""
    assert w.dim() >= 2 and w.is_contiguous()
    assert group_size in (32, 64, 128) and w.shape[-1] % group_size == 0, "group_size must be 32, 64 or 128 and divide K"
    code = _lib.dtype_code(w.dtype)
    _lib.require_cuda(w)
    k = w.shape[-1]
    lead = w.shape[:-1]
    q = w.new_empty(lead + (k // 2,), dtype=torch.uint8)
    scale = w.new_empty(lead + (k // group_size,))
    zero = None if symmetric else w.new_empty(lead + (k // group_size,), dtype=torch.uint8)
    with _lib.on_device(w.device):
        rc = _lib.load().b200quant_w4_group(_lib.ptr(w), _lib.ptr(q), _lib.ptr(scale),
                                            _lib.ptr(zero) if zero is not None else None, lead.numel(), k, group_size, code,
                                            _lib.stream_ptr(w.device))
    _lib.check(rc, "b200quant_w4_group")
    return q, scale, zero
