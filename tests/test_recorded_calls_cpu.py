"""Calls that somebody records - forward mode, jit traces, reverse mode - are recorded or refused, whether or not an operand
requires a gradient.  The kernels are replaced by fills of the output's memory, which autograd does not see either."""

import ctypes
import warnings

import pytest
import torch
from torch.autograd import forward_ad

from triton_grouped_gemm_b200 import _lib
from triton_grouped_gemm_b200.ep.autograd import combine_rows, permute_rows
from triton_grouped_gemm_b200.gemm import autograd as gemm_autograd
from triton_grouped_gemm_b200.gemm.autograd import grouped_gated_ffn
from triton_grouped_gemm_b200.gemm.BF16 import m_grouped_gated_gemm as gated_module
from triton_grouped_gemm_b200.gemm.BF16.m_grouped_gated_gemm import m_grouped_gated_gemm
from triton_grouped_gemm_b200.gemm.W4.m_grouped_gemm_w4 import m_grouped_gemm_w4, m_grouped_gemm_w4_gated

BF = torch.bfloat16
COUNT = torch.zeros(1, dtype=torch.int64)     # calls so far: what the fake kernels fill in


class _FakeLibrary:
    """Every entry point writes the number of the call, as bf16, into its output's first 64 values."""

    def __init__(self, outputs):
        self.outputs = outputs

    def __getattr__(self, name):
        def call(*args):
            if name == "b200gemm_gated_exponent_bytes":
                return 2 * args[0] * ((args[1] + 255) // 256 * 8)
            COUNT.add_(1)
            value = torch.full((64,), float(COUNT), dtype=BF)
            for i in self.outputs[name]:
                ctypes.memmove(args[i], value.data_ptr(), 128)
            return 0

        return call


@pytest.fixture(autouse=True)
def fake_device(monkeypatch):
    COUNT.zero_()
    lib = _FakeLibrary({"b200moe_permute_rows": [3], "b200moe_combine_rows": [4], "b200gemm_m_grouped_gated": [2],
                        "b200gemm_w4_m_grouped": [4], "b200gemm_m_grouped": [2]})
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)
    monkeypatch.setattr(_lib, "on_device", lambda d: _lib._no_guard)
    monkeypatch.setattr(_lib, "stream_ptr", lambda d: 0)
    monkeypatch.setattr(gemm_autograd, "_m_grouped_gemm_launch", lambda a, b, c, *rest: _lib.load().b200gemm_m_grouped(
        0, 0, c.data_ptr()))
    assert gated_module._lib is _lib


S = torch.tensor([2, 2])
POS = torch.arange(4)
W4 = (torch.zeros(2, 32, 16, dtype=torch.uint8), torch.ones(2, 32, 1, dtype=BF), None)
CALLS = {
    "permute_rows": (lambda x: permute_rows(x, POS, POS, 1), lambda: torch.randn(4, 16).to(BF)),
    "combine_rows": (lambda x: combine_rows(x, torch.ones(4, 1), POS, POS), lambda: torch.randn(4, 16).to(BF)),
    "combine_weights": (lambda w: combine_rows(torch.ones(4, 16, dtype=BF), w, POS, POS), lambda: torch.rand(4, 1)),
    "grouped_gated_ffn": (lambda x: grouped_gated_ffn(x, torch.ones(2, 32, 16, dtype=BF), torch.ones(2, 16, 16, dtype=BF), S),
                          lambda: torch.randn(4, 16).to(BF)),
    "m_grouped_gated_gemm": (lambda x: m_grouped_gated_gemm(x, torch.ones(2, 32, 16, dtype=BF), S), lambda: torch.randn(4, 16).to(BF)),
    "m_grouped_gemm_w4": (lambda x: m_grouped_gemm_w4(x, W4, S), lambda: torch.randn(4, 32).to(BF)),
    "m_grouped_gemm_w4_gated": (lambda x: m_grouped_gemm_w4_gated(x, W4, S), lambda: torch.randn(4, 32).to(BF)),
}
NO_GRADIENT = ["m_grouped_gated_gemm", "m_grouped_gemm_w4", "m_grouped_gemm_w4_gated"]


@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused(name):
    call, make = CALLS[name]
    x = make()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="jvp"):
            call(dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp"):
            call(dual)
        assert call(x).flatten()[0] > 0            # an operand without a tangent runs as ever


@pytest.mark.parametrize("name", CALLS)
def test_a_trace_runs_the_kernel_again(name):
    call, make = CALLS[name]
    x = make()
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        traced = torch.jit.trace(call, (x,), check_trace=False)
    before = int(COUNT)
    out = traced(x)
    assert int(COUNT) > before and float(out.flatten()[0]) == float(COUNT)
    before = int(COUNT)
    assert float(traced(x).flatten()[0]) > before


@pytest.mark.parametrize("name", CALLS)
def test_make_fx_is_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx

    call, make = CALLS[name]
    with pytest.raises(RuntimeError, match="cannot be traced by make_fx"):
        make_fx(call)(make())


@pytest.mark.parametrize("name", CALLS)
def test_reverse_mode(name):
    call, make = CALLS[name]
    x = make().requires_grad_()
    y = call(x)
    assert y.requires_grad
    if name in NO_GRADIENT:
        with pytest.raises(RuntimeError, match="no gradient"):
            y.float().sum().backward()
    with torch.no_grad():
        assert not call(x).requires_grad
    with torch.inference_mode():
        assert not call(x.detach()).requires_grad


@pytest.mark.parametrize("name", ["m_grouped_gated_gemm", "m_grouped_gemm_w4"])
def test_out_is_outside_autograd_and_refused_where_that_goes_unnoticed(name):
    if name == "m_grouped_gated_gemm":
        x, out = torch.randn(4, 16).to(BF), torch.zeros(4, 16, dtype=BF)
        call = lambda x: m_grouped_gated_gemm(x, torch.ones(2, 32, 16, dtype=BF), S, out=out)  # noqa: E731
    else:
        x, out = torch.randn(4, 32).to(BF), torch.zeros(4, 32, dtype=BF)
        call = lambda x: m_grouped_gemm_w4(x, W4, S, out=out)  # noqa: E731
    assert call(x) is out and call(x.detach().requires_grad_()) is out and not out.requires_grad
    with forward_ad.dual_level():
        assert call(x) is out
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, (x,), check_trace=False)
