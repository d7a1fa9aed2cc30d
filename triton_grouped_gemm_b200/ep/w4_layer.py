"""MoE feed-forward layer with 4-bit expert weights for decoding on one rank: a quarter of the 16-bit weights' bytes
(half of FP8's) per step, which is what a step with few tokens costs."""

from __future__ import annotations

import torch

from ..gemm.W4.m_grouped_gemm_w4 import m_grouped_gemm_w4, m_grouped_gemm_w4_gated
from ..quant.per_group_cast import per_group_cast_to_w4
from .autograd import check_routing, combine_rows, permute_rows
from .dispatch import make_plan


class W4MoELayer:
    def __init__(self, w13: torch.Tensor, w2: torch.Tensor, group_size: int = 128, symmetric: bool = True,
                 activation: str = "silu"):
        """w13 [E, 2*I, H] (gate rows, then up rows), w2 [E, H, I], bf16 or fp16; quantised once here.  H and I are
        multiples of ``group_size`` (32, 64 or 128)."""
        assert w13.dim() == 3 and w2.dim() == 3 and w2.shape == (w13.shape[0], w13.shape[2], w13.shape[1] // 2)
        self.num_experts = w13.shape[0]
        self.activation = activation
        self.w13 = per_group_cast_to_w4(w13.detach().contiguous(), group_size, symmetric)
        self.w2 = per_group_cast_to_w4(w2.detach().contiguous(), group_size, symmetric)

    @torch.no_grad()
    def forward(self, x: torch.Tensor, topk_idx: torch.Tensor, topk_weight: torch.Tensor) -> torch.Tensor:
        """x [T, H] of the weights' type, topk_idx / topk_weight [T, k] -> [T, H].  A pair whose expert id is out of
        range is dropped.  Runs under ``no_grad``: the result is detached."""
        check_routing("W4MoELayer", x, topk_idx, topk_weight)
        plan = make_plan(topk_idx, self.num_experts)
        rows = permute_rows(x, plan.pos, plan.send_order, plan.top_k)
        h = m_grouped_gemm_w4_gated(rows, self.w13, plan.size_per_group, self.activation)
        y = m_grouped_gemm_w4(h, self.w2, plan.size_per_group)
        return combine_rows(y, topk_weight, plan.pos, plan.send_order)

    __call__ = forward
