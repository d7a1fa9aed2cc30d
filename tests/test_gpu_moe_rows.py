"""Permute and combine with their gradients, and the trainable and the 4-bit MoE layer made of the operators."""

import pytest
import torch

from gated_ffn_ref import HALF_EPS, HALF_TINY, assert_within, block
from triton_grouped_gemm_b200 import _lib
from triton_grouped_gemm_b200.ep.autograd import combine_rows, moe_ffn, permute_rows
from triton_grouped_gemm_b200.ep.dispatch import make_plan
from triton_grouped_gemm_b200.ep.w4_layer import W4MoELayer

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _plan(t, k, experts, seed, drop=0.0):
    gen = torch.Generator().manual_seed(seed)
    idx = torch.stack([torch.randperm(experts, generator=gen)[:k] for _ in range(t)]) if t else torch.zeros(0, k, dtype=torch.int64)
    idx[torch.rand(t, k, generator=gen) < drop] = -1
    plan = make_plan(idx.to(DEV), experts)
    return idx, plan


def _rounded(value, magnitude, terms, dtype):
    """(value, bound): `terms` fp32 multiply-adds (2^-24 each of the magnitudes), one rounding."""
    e = (terms + 1) * 2.0 ** -24 * magnitude
    return value, e + HALF_EPS[dtype] * (value.abs() + e) + HALF_TINY[dtype]


def _reference(x, rows, w, drows, dout, pos, order, t, k):
    """Plain 64-bit forms by index arithmetic over the pairs that own their row."""
    h, r = x.shape[1], order.numel()
    pairs = torch.arange(t * k, device=DEV)
    inside = (pos >= 0) & (pos < r)
    owns = inside & (order[pos.clamp(0, max(r - 1, 0))] == pairs) if r else torch.zeros_like(inside)
    token, at = (pairs // k)[owns], pos[owns]
    wp = w.double().reshape(-1)[owns].unsqueeze(1)
    z = lambda n: torch.zeros(n, h, device=DEV, dtype=torch.float64)  # noqa: E731
    perm = z(r).index_copy_(0, at, x.double()[token])
    dx, mdx = (z(t).index_add_(0, token, v) for v in (drows.double()[at], drows.double()[at].abs()))
    out, mout = (z(t).index_add_(0, token, v) for v in (rows.double()[at] * wp, (rows.double()[at] * wp).abs()))
    dr = z(r).index_copy_(0, at, dout.double()[token] * wp)
    dw, mdw = torch.zeros(t * k, device=DEV, dtype=torch.float64), torch.zeros(t * k, device=DEV, dtype=torch.float64)
    prod = dout.double()[token] * rows.double()[at]
    dw[owns], mdw[owns] = prod.sum(1), prod.abs().sum(1)
    dtype = x.dtype
    return dict(perm=perm, dx=_rounded(dx, mdx, k, dtype), out=_rounded(out, mout, k, dtype), dr=_rounded(dr, dr.abs(), 1, dtype),
                dw=(dw.view(t, k), ((h + 40) * 2.0 ** -24 * mdw + 1e-44).view(t, k)))


def _check(t, k, hidden, dtype, pos, order, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(dtype)  # noqa: E731
    r = order.numel()
    x, rows, drows, dout = n(t, hidden), n(r, hidden), n(r, hidden), n(t, hidden)
    w = torch.rand(t, k, generator=gen, device=DEV)
    ref = _reference(x, rows, w, drows, dout, pos, order, t, k)
    x.requires_grad_()
    got = permute_rows(x, pos, order, k)
    assert torch.equal(got.double(), ref["perm"])
    assert_within(torch.autograd.grad(got, x, drows)[0], ref["dx"], "dx")
    rows.requires_grad_()
    w.requires_grad_()
    out = combine_rows(rows, w, pos, order)
    assert_within(out, ref["out"], "out")
    dr, dw = torch.autograd.grad(out, (rows, w), dout)
    assert_within(dr, ref["dr"], "drows")
    assert_within(dw, ref["dw"], "dweight")
    with torch.no_grad():
        assert torch.equal(permute_rows(x, pos, order, k), got) and torch.equal(combine_rows(rows, w, pos, order), out)
    # each gradient alone
    assert torch.equal(torch.autograd.grad(combine_rows(rows, w.detach(), pos, order), rows, dout)[0], dr)
    assert torch.equal(torch.autograd.grad(combine_rows(rows.detach(), w, pos, order), w, dout)[0], dw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,k,hidden", [(1, 1, 8), (1, 8, 4096), (5, 3, 72), (333, 2, 1032), (64, 9, 136), (40, 32, 24),
                                        (3000, 4, 264), (2500, 8, 1000), (9000, 1, 8), (2600, 17, 32)])
def test_rows_and_gradients(t, k, hidden, dtype):
    _, plan = _plan(t, k, 48, seed=t + k)
    assert _lib.device_status() == 0
    _check(t, k, hidden, dtype, plan.pos, plan.send_order)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("t", [50, 3000])
def test_dropped_pairs(t):
    _, plan = _plan(t, 4, 16, seed=3, drop=0.3)
    _lib.device_status()
    _check(t, 4, 136, torch.bfloat16, plan.pos, plan.send_order)
    assert _lib.device_status() == 0x20


def test_all_pairs_dropped_and_no_tokens():
    pos = torch.full((6,), -1, device=DEV)
    _check(3, 2, 16, torch.bfloat16, pos, pos)
    assert _lib.device_status() == 0x20
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    _check(0, 2, 16, torch.bfloat16, none, none)
    _check(0, 2, 16, torch.bfloat16, none, torch.full((5,), -1, device=DEV))      # rows without tokens: zeros
    assert _lib.device_status() == 0


def test_bad_plans_touch_nothing_out_of_bounds():
    """Rows out of range, a row named twice, an order that contradicts pos: such pairs take no part, whoever they are."""
    t, k = 200, 2
    pos = torch.randperm(t * k, device=DEV)
    order = torch.empty_like(pos)
    order[pos] = torch.arange(t * k, device=DEV)
    pos[3], pos[4], pos[5], pos[6] = t * k, -7, 2 ** 40, -(2 ** 62)
    pos[10] = pos[11]
    order[20:24] = torch.tensor([t * k, -2, 2 ** 50, 0], device=DEV)
    _check(t, k, 72, torch.float16, pos, order)
    assert _lib.device_status() == 0x20
    _check(t, k, 72, torch.float16, pos, order[:150].contiguous())                # fewer rows than pairs
    more = torch.cat([order, torch.full((300,), -1, device=DEV)])                 # more rows than pairs
    _check(t, k, 72, torch.float16, pos, more)
    assert _lib.device_status() == 0x20


def test_weights_in_16_bits_and_views():
    _, plan = _plan(30, 2, 8, seed=1)
    rows = torch.randn(60, 64, device=DEV).bfloat16()
    w = torch.rand(2, 30, device=DEV).bfloat16().t().requires_grad_()             # a strided weight matrix
    out = combine_rows(rows, w, plan.pos, plan.send_order)
    out.sum().backward()                                                          # a gradient with strides of zero
    assert w.grad.dtype == torch.bfloat16 and w.grad.shape == (30, 2)
    want = rows.double().sum(1)[plan.pos].view(30, 2)
    assert_within(w.grad, _rounded(want, rows.double().abs().sum(1)[plan.pos].view(30, 2), 64, torch.bfloat16), "dweight")
    xt = torch.randn(64, 30, device=DEV).bfloat16().t().requires_grad_()
    got = permute_rows(xt, plan.pos, plan.send_order, 2)
    assert torch.equal(got, xt[plan.send_order // 2])


def test_second_derivatives_are_refused():
    _, plan = _plan(6, 2, 8, seed=1)
    x = torch.randn(6, 16, device=DEV).bfloat16().requires_grad_()
    rows = permute_rows(x, plan.pos, plan.send_order, 2)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(rows.sum(), x, create_graph=True)
    w = torch.rand(6, 2, device=DEV).requires_grad_()
    out = combine_rows(rows.detach(), w, plan.pos, plan.send_order)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(out.float().sum(), w, create_graph=True)
    w13, w2 = _layer(8, 16, 8, torch.bfloat16, 3)
    y = moe_ffn(x, torch.zeros(6, 1, dtype=torch.int64, device=DEV), torch.ones(6, 1, device=DEV), w13.requires_grad_(), w2)
    with pytest.raises(RuntimeError, match="differentiable once|differentiate twice"):
        torch.autograd.grad(torch.autograd.grad(y.float().sum(), w13, create_graph=True)[0].float().sum(), w13)


# ------------------------------------------------------------------------------------------- the operators together
def _layer(experts, hidden, inter, dtype, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n = lambda std, *s: (torch.randn(*s, generator=gen, device=DEV) * std).to(dtype)  # noqa: E731
    return n(hidden ** -0.5, experts, 2 * inter, hidden), n(inter ** -0.5, experts, hidden, inter)


@pytest.mark.parametrize("drop", [0.0, 0.2])
def test_trainable_layer(drop):
    """Forward and all four gradients against the layer written out in 64 bits.  Relative 2-norm: four roundings of bf16
    lie between input and output (rows' y, out) and up to five on a gradient's way (dy, dgu, dx of the rows, sum, and the
    kept h), each of relative 2-norm error at most 2^-8: 5 * 2^-8."""
    t, k, experts, hidden, inter = 150, 3, 8, 128, 96
    idx, _ = _plan(t, k, experts, seed=2, drop=drop)
    w13, w2 = _layer(experts, hidden, inter, torch.bfloat16, 4)
    x = torch.randn(t, hidden, device=DEV).bfloat16()
    w = torch.softmax(torch.randn(t, k, device=DEV), 1)
    dout = torch.randn(t, hidden, device=DEV).bfloat16()
    leaves = [v.detach().requires_grad_() for v in (x, w, w13, w2)]
    out = moe_ffn(leaves[0], idx.to(DEV), leaves[1], leaves[2], leaves[3])
    got = (out,) + torch.autograd.grad(out, leaves, dout)
    ref = [v.detach().double().requires_grad_() for v in (x, w, w13, w2)]
    total = torch.zeros(t, hidden, device=DEV, dtype=torch.float64)
    for e in range(experts):
        token, j = (idx == e).nonzero(as_tuple=True)
        gate, up = (ref[0][token] @ ref[2][e].t()).chunk(2, 1)
        y = (torch.nn.functional.silu(gate) * up) @ ref[3][e].t()
        total = total.index_add(0, token.to(DEV), y * ref[1][token, j].unsqueeze(1))
    want = (total,) + torch.autograd.grad(total, ref, dout.double())
    for a, b, name in zip(got, want, ("out", "dx", "dweight", "dw13", "dw2")):
        assert (a.double() - b).norm() <= 5 * 2.0 ** -8 * b.norm(), name
    assert _lib.device_status() == (0x20 if drop else 0)


def test_trainable_layer_captured_with_an_eager_graph_alive():
    """The layer's step captured into a graph while an eager step's autograd graph of the same parameters lives on.  The
    captured step differentiates leaves of its own (detached views of the same memory): torch ties a leaf's
    accumulation node to the stream of the graph that made it, and a capture may not wait for that stream."""
    t, k, experts, hidden, inter = 64, 2, 4, 64, 48
    idx, _ = _plan(t, k, experts, seed=6)
    idx = idx.to(DEV)
    w13, w2 = (v.requires_grad_() for v in _layer(experts, hidden, inter, torch.bfloat16, 7))
    x = torch.randn(t, hidden, device=DEV).bfloat16().requires_grad_()
    w = torch.softmax(torch.randn(t, k, device=DEV), 1).requires_grad_()
    params = (x, w, w13, w2)
    dout = torch.randn(t, hidden, device=DEV).bfloat16()

    def step():
        own = [v.detach().requires_grad_() for v in params]
        out = moe_ffn(own[0], idx, *own[1:])
        return (out.detach(),) + torch.autograd.grad(out, own, dout)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    alive = moe_ffn(x, idx, w, w13, w2)
    eager = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    graph.replay()
    torch.cuda.synchronize()

    def near(a, b):   # the routing plan's order inside an expert is free, so sums over its rows may differ in order
        return (a.double() - b.double()).norm() <= 2.0 ** -8 * b.double().norm()

    assert all(near(a, b) for a, b in zip(captured, eager))
    again = torch.autograd.grad(alive, params, dout)
    assert all(near(a, b) for a, b in zip(again, eager[1:]))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,drop", [(1, 0.0), (7, 0.0), (120, 0.1)])
def test_w4_layer(t, drop, dtype, symmetric):
    """Against the layer with the quantised weights' values in 64 bits: roundings of h, y and out, each at most eps/2 in
    relative 2-norm, and 2^-12 for the fp32 sums."""
    k, experts, hidden, inter, gs = 4, 16, 256, 192, 64
    idx, _ = _plan(t, k, experts, seed=t, drop=drop)
    layer = W4MoELayer(*_layer(experts, hidden, inter, dtype, 9), group_size=gs, symmetric=symmetric)
    x = torch.randn(t, hidden, device=DEV).to(dtype)
    w = torch.softmax(torch.randn(t, k, device=DEV), 1)
    got = layer(x, idx.to(DEV), w)

    def values(b):
        whole = torch.stack((b[0] & 15, b[0] >> 4), -1).flatten(-2).double()
        z = 8.0 if b[2] is None else b[2].double().repeat_interleave(gs, -1)
        return (whole - z) * b[1].double().repeat_interleave(gs, -1)

    w13, w2 = values(layer.w13), values(layer.w2)
    want = torch.zeros(t, hidden, device=DEV, dtype=torch.float64)
    for e in range(experts):
        token, j = (idx == e).nonzero(as_tuple=True)
        gate, up = (x[token].double() @ w13[e].t()).chunk(2, 1)
        y = (torch.nn.functional.silu(gate) * up) @ w2[e].t()
        want.index_add_(0, token.to(DEV), y * w[token, j].double().unsqueeze(1))
    assert (got.double() - want).norm() <= (3 * HALF_EPS[dtype] + 2.0 ** -12) * want.norm()
    _lib.device_status()


def test_block_reference_is_what_autograd_says():
    """The written-out gradients that the other tests lean on, against differentiating the forward in 64 bits."""
    sizes, hidden, inter = [9, 0, 4], 24, 16
    gen = torch.Generator(device=DEV).manual_seed(1)
    n = lambda *s: torch.randn(*s, generator=gen, device=DEV).bfloat16()  # noqa: E731
    x, w13, w2, dy = n(13, hidden), n(3, 2 * inter, hidden), n(3, hidden, inter), n(13, hidden)
    for act, f in (("silu", torch.nn.functional.silu), ("gelu_tanh", lambda v: torch.nn.functional.gelu(v, approximate="tanh"))):
        ref = block(x, w13, w2, sizes, act, dy)
        leaves = [v.double().requires_grad_() for v in (x, w13, w2)]
        ys = [(lambda gu: f(gu[0]) * gu[1])((xe @ leaves[1][e].t()).chunk(2, 1)) @ leaves[2][e].t()
              for e, xe in enumerate(leaves[0].split(sizes))]
        grads = torch.autograd.grad(torch.cat(ys), leaves, dy.double())
        for a, name in zip(grads, ("dx", "dw13", "dw2")):
            assert (a - ref[name][0]).norm() <= 1e-12 * a.norm()
