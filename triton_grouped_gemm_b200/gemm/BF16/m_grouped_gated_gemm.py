"""BF16 / FP16 M-grouped GEMM of a gated feed-forward block: gate and up projection, activation and product
in one kernel.

``H[rows of g] = act(A[rows of g] @ Wg_g.T) * (A[rows of g] @ Wu_g.T)`` with fp32 accumulation and one rounding;
``B`` [G, 2*I, K] holds the gate rows, then the up rows.  The reference leaves the activation to separate torch
steps between two grouped GEMMs (README.md:175-179).  ``gemm.autograd.grouped_gated_ffn`` is the whole block with
its gradients.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from ... import _lib

ACTIVATIONS = {"silu": 0, "gelu_tanh": 1}


def activation_code(activation: str) -> int:
    code = ACTIVATIONS.get(activation, -1)
    assert code >= 0, f"activation {activation!r} not supported; expected one of: {', '.join(ACTIVATIONS)}"
    return code


def _check(A: Tensor, B: Tensor, size_per_group: Tensor) -> Tuple[int, int, int, int]:
    assert A.dim() == 2, "A must be 2D [M, K]"
    assert B.dim() == 3, "B must be 3D [num_groups, 2*I, K]"
    m, k = A.shape
    g, two_i, bk = B.shape
    assert bk == k, "K of A should be equal to K of B"
    assert two_i % 2 == 0, "B must hold as many gate rows as up rows"
    inter = two_i // 2
    assert B.dtype == A.dtype, "A and B must share one dtype"
    assert (k * A.element_size()) % 16 == 0, "TMA required 16-byte alignment"
    assert (inter * A.element_size()) % 16 == 0, "TMA required 16-byte alignment"
    assert A.is_contiguous() and B.is_contiguous(), "A and B must be contiguous"
    assert size_per_group.numel() == g, "size_per_group must have one entry per group"
    _lib.require_cuda(A, B, size_per_group)
    assert A.device == B.device == size_per_group.device, "A, B and size_per_group must be on one device"
    return m, k, g, inter


def _m_grouped_gated_launch(A: Tensor, B: Tensor, size_per_group: Tensor, activation: str, *, out: Optional[Tensor] = None,
                            save: bool = False, masked_stride: int = 0, tail: Optional[Tensor] = None,
                            numSM: int = -1) -> Tuple[Tensor, Optional[Tensor], Optional[Tensor]]:
    """(h, saved codes, saved exponents); the saved pair (None without ``save``) is what
    ``_m_grouped_gated_grad_launch`` takes.  ``tail``: [M, *] matrix whose rows behind the last group are zeroed."""
    code = _lib.dtype_code(A.dtype)
    act = activation_code(activation)
    m, k, g, inter = _check(A, B, size_per_group)
    if masked_stride:
        assert m == g * masked_stride, "A must hold masked_stride rows per group"
    lib = _lib.load()
    h = A.new_empty(m, inter) if out is None else out
    assert h.shape == (m, inter) and h.dtype == A.dtype and h.is_contiguous() and h.device == A.device, \
        "out should be contiguous, of A's type and device and of shape [M, I]"
    saved = exps = None
    if save:
        saved = A.new_empty(m, 2 * inter, dtype=torch.int16)
        exps = A.new_empty(lib.b200gemm_gated_exponent_bytes(m, inter), dtype=torch.uint8)
    sizes, is64 = _lib.sizes_arg(size_per_group)
    with _lib.on_device(A.device):
        rc = lib.b200gemm_m_grouped_gated(
            _lib.ptr(A), _lib.ptr(B), _lib.ptr(h), _lib.ptr(saved) if save else None, _lib.ptr(exps) if save else None,
            _lib.ptr(sizes), is64, g, m, int(masked_stride), inter, k, act, code,
            _lib.ptr(tail) if tail is not None else None, tail.shape[1] if tail is not None else 0, int(numSM),
            _lib.stream_ptr(A.device))
    _lib.check(rc, "b200gemm_m_grouped_gated")
    return h, saved, exps


def _m_grouped_gated_grad_launch(dY: Tensor, W2: Tensor, saved: Tensor, exps: Tensor, size_per_group: Tensor,
                                 activation: str, tail: Optional[Tensor] = None, numSM: int = -1) -> Tensor:
    """[M, 2*I] gradient of the gate and up products: dH = dY @ W2_g (W2 [G, K, I]) and the gate's derivative in
    one kernel."""
    m, k = dY.shape
    g, wk, inter = W2.shape
    assert wk == k and saved.shape == (m, 2 * inter) and dY.is_contiguous() and W2.is_contiguous()
    assert dY.dtype == W2.dtype and size_per_group.numel() == g
    dgu = dY.new_empty(m, 2 * inter)
    sizes, is64 = _lib.sizes_arg(size_per_group)
    with _lib.on_device(dY.device):
        rc = _lib.load().b200gemm_m_grouped_gated_grad(
            _lib.ptr(dY), _lib.ptr(W2), _lib.ptr(saved), _lib.ptr(exps), _lib.ptr(dgu), _lib.ptr(sizes), is64, g, m, inter, k,
            activation_code(activation), _lib.dtype_code(dY.dtype), _lib.ptr(tail) if tail is not None else None,
            tail.shape[1] if tail is not None else 0, int(numSM), _lib.stream_ptr(dY.device))
    _lib.check(rc, "b200gemm_m_grouped_gated_grad")
    return dgu


class _MGroupedGatedGemm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, A, B, size_per_group, activation, masked_stride, numSM):
        return _m_grouped_gated_launch(A, B, size_per_group, activation, masked_stride=masked_stride, numSM=numSM)[0]

    @staticmethod
    def backward(ctx, dh):
        raise RuntimeError("m_grouped_gated_gemm has no gradient; grouped_gated_ffn is the block with one")


def m_grouped_gated_gemm(A: Tensor, B: Tensor, size_per_group: Tensor, activation: str = "silu", *,
                         masked_stride: int = 0, out: Optional[Tensor] = None, numSM: int = -1) -> Tensor:
    """[M, I] of A [M, K], B [G, 2*I, K] (gate rows, then up rows); ``activation`` "silu" or "gelu_tanh".
    K and I are multiples of 8.  ``masked_stride`` > 0: masked row layout (``masked_stride`` rows per group, the
    first ``size_per_group[g]`` of them valid).  Rows outside the groups are left as they were in ``out``.  No
    gradient (differentiating through the result raises; ``out`` is written outside autograd): see
    ``gemm.autograd.grouped_gated_ffn``."""
    if out is not None:
        _lib.refuse_recorded_out("m_grouped_gated_gemm", A, B)
    elif _lib.recorded("m_grouped_gated_gemm", A, B):
        return _MGroupedGatedGemm.apply(A, B, size_per_group, activation, masked_stride, numSM)
    return _m_grouped_gated_launch(A, B, size_per_group, activation, out=out, masked_stride=masked_stride, numSM=numSM)[0]
