"""Differentiable row movement between tokens and experts on one rank, and the trainable MoE layer made of it.

``pos`` (row of pair p = t * top_k + j) and ``order`` (pair of row r) are the two halves of a routing plan:
``make_plan(topk_idx, num_experts)`` gives them as ``plan.pos`` and ``plan.send_order``.  A pair whose ``pos`` is
out of range (the -1 of a dropped token) or whose row's ``order`` names another pair takes no part and raises
status bit ``0x20``; a row that no pair owns reads as zeros.  For 16-bit rows on one rank these are the ones to use.
``ep.dispatch.dispatch`` / ``combine`` move payloads of any type, also between ranks, forward only (81 920 tokens, top-8,
hidden 2048 on one rank: permute 0.51 ms here, 0.82 there; combine 0.47 and 0.48); the reference has these operators only in its vendored baseline (grouped_gemm/ops.py permute /
unpermute).
"""

from __future__ import annotations

import torch

from .. import _lib
from ..gemm.autograd import grouped_gated_ffn
from .dispatch import make_plan


def _check_plan(what: str, rows: torch.Tensor, pos: torch.Tensor, order: torch.Tensor, pairs: int) -> None:
    assert rows.dtype in (torch.bfloat16, torch.float16), f"{what}: data type {rows.dtype} not supported"
    assert pos.dtype == torch.int64 and order.dtype == torch.int64, f"{what}: pos and order must be int64"
    assert pos.numel() == pairs and pos.is_contiguous() and order.is_contiguous() and order.dim() == 1, \
        f"{what}: pos must hold one contiguous entry per (token, k) pair and order one per row"
    _lib.require_cuda(rows, pos, order)
    device = rows.get_device()
    assert pos.get_device() == device and order.get_device() == device, f"{what}: all operands must be on one device"


def _once(what: str) -> None:
    # autograd calls backward with gradients enabled only to differentiate it again, which these kernels cannot
    # (cheaper than once_differentiable's wrapper, 3 us of a call)
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} is differentiable once: create_graph=True is not supported")


def _permute(x, pos, order, top_k):
    t, h = x.shape
    out = x.new_empty(order.numel(), h)
    with _lib.on_device(x.device):
        rc = _lib.load().b200moe_permute_rows(x.data_ptr(), pos.data_ptr(), order.data_ptr(), out.data_ptr(), t, top_k, h,
                                              order.numel(), _lib.stream_ptr(x.device))
    _lib.check(rc, "b200moe_permute_rows")
    return out


def _combine(rows, w32, pos, order, tokens, top_k):
    r, h = rows.shape
    out = rows.new_empty(tokens, h)
    with _lib.on_device(rows.device):
        rc = _lib.load().b200moe_combine_rows(rows.data_ptr(), pos.data_ptr(), order.data_ptr(),
                                              w32.data_ptr() if w32 is not None else None, out.data_ptr(), tokens, top_k, h, r,
                                              _lib.dtype_code(rows.dtype), _lib.stream_ptr(rows.device))
    _lib.check(rc, "b200moe_combine_rows")
    return out


class _PermuteRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, order, top_k):
        ctx.save_for_backward(pos, order)
        ctx.top_k = top_k
        return _permute(x, pos, order, top_k)

    @staticmethod
    def backward(ctx, drows):
        _once("permute_rows")
        pos, order = ctx.saved_tensors
        return _combine(_lib.aligned(drows), None, pos, order, pos.numel() // ctx.top_k, ctx.top_k), None, None, None


class _CombineRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, topk_weight, pos, order):
        t, top_k = topk_weight.shape
        w32 = topk_weight.to(torch.float32).contiguous()
        ctx.save_for_backward(rows if ctx.needs_input_grad[1] else None, w32, pos, order)
        ctx.num_rows, ctx.weight_dtype = rows.shape[0], topk_weight.dtype
        return _combine(rows, w32, pos, order, t, top_k)

    @staticmethod
    def backward(ctx, dout):
        _once("combine_rows")
        rows, w32, pos, order = ctx.saved_tensors
        dout = _lib.aligned(dout)
        t, h = dout.shape
        drows = dout.new_empty(ctx.num_rows, h) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(w32) if ctx.needs_input_grad[1] else None
        with _lib.on_device(dout.device):
            rc = _lib.load().b200moe_combine_rows_grad(
                dout.data_ptr(), rows.data_ptr() if rows is not None else None, pos.data_ptr(), order.data_ptr(),
                w32.data_ptr(), drows.data_ptr() if drows is not None else None, dw.data_ptr() if dw is not None else None,
                t, w32.shape[1], h, ctx.num_rows, _lib.dtype_code(dout.dtype), _lib.stream_ptr(dout.device))
        _lib.check(rc, "b200moe_combine_rows_grad")
        return drows, dw.to(ctx.weight_dtype) if dw is not None else None, None, None


def permute_rows(x: torch.Tensor, pos: torch.Tensor, order: torch.Tensor, top_k: int) -> torch.Tensor:
    """x [T, H] bf16 / fp16 -> rows [R, H] with ``rows[pos[t * top_k + j]] = x[t]`` (R = order.numel()), differentiable
    in x.  H a multiple of 8, top_k <= 32."""
    assert x.dim() == 2, "x must be 2D [T, H]"
    _check_plan("permute_rows", x, pos, order, x.shape[0] * top_k)
    x = x.contiguous()
    if _lib.recorded("permute_rows", x):
        return _PermuteRows.apply(x, pos, order, top_k)
    return _permute(x, pos, order, top_k)


def combine_rows(rows: torch.Tensor, topk_weight: torch.Tensor, pos: torch.Tensor, order: torch.Tensor) -> torch.Tensor:
    """rows [R, H] bf16 / fp16, topk_weight [T, k] -> [T, H] with ``out[t] = sum_j topk_weight[t, j] *
    rows[pos[t * k + j]]`` (fp32 weights and sums, whatever topk_weight's type), differentiable in rows and topk_weight.  H a multiple of 8, k <= 32."""
    assert rows.dim() == 2 and topk_weight.dim() == 2, "rows must be 2D [R, H] and topk_weight 2D [T, k]"
    assert topk_weight.is_floating_point(), "topk_weight must be floating point"
    assert order.numel() == rows.shape[0], "order must have one entry per row"
    _check_plan("combine_rows", rows, pos, order, topk_weight.numel())
    assert topk_weight.get_device() == rows.get_device(), "combine_rows: all operands must be on one device"
    rows = rows.contiguous()
    if _lib.recorded("combine_rows", rows, topk_weight):
        return _CombineRows.apply(rows, topk_weight, pos, order)
    t, top_k = topk_weight.shape
    return _combine(rows, topk_weight.to(torch.float32).contiguous(), pos, order, t, top_k)


def check_routing(what: str, x: torch.Tensor, topk_idx: torch.Tensor, topk_weight: torch.Tensor) -> None:
    assert x.dim() == 2 and topk_idx.dim() == 2 and topk_idx.shape[0] == x.shape[0], \
        f"{what}: x must be 2D [T, H] and topk_idx 2D [T, k]"
    assert topk_weight.shape == topk_idx.shape, f"{what}: topk_weight must have topk_idx's shape"


def moe_ffn(x: torch.Tensor, topk_idx: torch.Tensor, topk_weight: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor,
            activation: str = "silu") -> torch.Tensor:
    """Trainable 16-bit MoE feed-forward layer on one rank: x [T, H], topk_idx [T, k] (an id outside the experts drops
    the pair), topk_weight [T, k], w13 [E, 2*I, H] (gate rows, then up rows), w2 [E, H, I] -> [T, H], with gradients
    for x, topk_weight, w13 and w2.  Nothing synchronises the host (up to 1024 experts).  The plan leaves the order of the rows inside an
    expert open: it changes nothing in the output or the gradients of x and topk_weight, but the weights' gradients sum
    over the rows and may differ in their last bits from one call to the next."""
    check_routing("moe_ffn", x, topk_idx, topk_weight)
    top_k = topk_idx.shape[1]
    plan = make_plan(topk_idx, w13.shape[0])
    rows = permute_rows(x, plan.pos, plan.send_order, top_k)
    y = grouped_gated_ffn(rows, w13, w2, plan.size_per_group, activation)
    return combine_rows(y, topk_weight, plan.pos, plan.send_order)
