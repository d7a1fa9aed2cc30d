"""The grouped kernels may be set up while their predecessor in the stream drains: results of launches queued back to
back, where each reads what the one before wrote, have to be those of launches with the device idle in between."""

import pytest
import torch

from triton_grouped_gemm_b200 import _lib
from triton_grouped_gemm_b200.ep.autograd import combine_rows, permute_rows
from triton_grouped_gemm_b200.gemm.autograd import grouped_gated_ffn
from triton_grouped_gemm_b200.gemm.BF16.k_grouped_gemm_TMA import k_grouped_gemm
from triton_grouped_gemm_b200.gemm.BF16.m_grouped_gemm_TMA import m_grouped_gemm
from triton_grouped_gemm_b200.gemm.W4.m_grouped_gemm_w4 import m_grouped_gemm_w4, m_grouped_gemm_w4_gated
from triton_grouped_gemm_b200.quant.per_group_cast import per_group_cast_to_w4

pytestmark = pytest.mark.gpu


def _problem(tokens, experts, hidden, inter, top_k):
    gen = torch.Generator(device="cuda").manual_seed(7)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(std).to(torch.bfloat16)

    expert = torch.topk(torch.rand(tokens, experts, generator=gen, device="cuda"), top_k, dim=1).indices.reshape(-1)
    order = torch.argsort(expert, stable=True)
    pos = torch.empty_like(order)
    pos[order] = torch.arange(order.numel(), device="cuda")
    sizes = torch.bincount(expert, minlength=experts)
    w13, w2 = normal(experts, 2 * inter, hidden, std=hidden ** -0.5), normal(experts, hidden, inter, std=inter ** -0.5)
    weight = torch.softmax(torch.rand(tokens, top_k, generator=gen, device="cuda"), 1)
    return normal(tokens, hidden), weight, order, pos, sizes, w13, w2


def _steps(problem, top_k, pause, layers=6):
    """A few layers forward, one of them 4-bit, with a weight gradient each; ``pause()`` between any two calls."""
    x, weight, order, pos, sizes, w13, w2 = problem
    g13, g2 = per_group_cast_to_w4(w13, 64), per_group_cast_to_w4(w2, 64, symmetric=False)
    pause()
    kept = []
    for layer in range(layers):
        rows = permute_rows(x, pos, order, top_k)
        pause()
        if layer % 3 == 1:
            h = m_grouped_gemm_w4_gated(rows, g13, sizes)
            pause()
            y = m_grouped_gemm_w4(h, g2, sizes)
        elif layer % 3 == 2:
            c = m_grouped_gemm(rows, w13, sizes, trans_b=True)
            pause()
            y = m_grouped_gemm(c, w13, sizes, trans_b=False)
        else:
            y = grouped_gated_ffn(rows, w13, w2, sizes)
        pause()
        kept.append(k_grouped_gemm(y, rows, sizes))
        pause()
        x = combine_rows(y, weight, pos, order)
        pause()
        kept.append(x)
    return kept


@pytest.mark.parametrize("tokens,experts,hidden,inter,top_k", [
    (1, 16, 256, 128, 4),          # launches shorter than their setup
    (37, 16, 512, 256, 2),
    (600, 8, 1024, 512, 4),
    (4096, 4, 1024, 512, 2),       # CTA pairs
])
def test_back_to_back_as_one_by_one(tokens, experts, hidden, inter, top_k):
    problem = _problem(tokens, experts, hidden, inter, top_k)
    want = _steps(problem, top_k, torch.cuda.synchronize)
    for _ in range(10):
        got = _steps(problem, top_k, lambda: None)
        for g, w in zip(got, want):
            assert torch.equal(g, w)
    assert _lib.device_status() == 0


def test_replayed_and_across_streams():
    problem = _problem(37, 16, 512, 256, 2)
    want = _steps(problem, 2, torch.cuda.synchronize)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _steps(problem, 2, lambda: None)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _steps(problem, 2, lambda: None)
    for _ in range(5):
        for g in got:
            g.zero_()
        graph.replay()
        graph.replay()
        for g, w in zip(got, want):
            assert torch.equal(g, w)

    # every call on the other of two streams, ordered by events
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    turn = [0]
    main = torch.cuda.current_stream()

    def hand_over():
        now, turn[0] = streams[turn[0]], 1 - turn[0]
        streams[turn[0]].wait_stream(now)
        torch.cuda.set_stream(streams[turn[0]])

    try:
        streams[0].wait_stream(main)
        torch.cuda.set_stream(streams[0])
        got = _steps(problem, 2, hand_over)
        torch.cuda.synchronize()
    finally:
        torch.cuda.set_stream(main)
    for g, w in zip(got, want):
        assert torch.equal(g, w)
    assert _lib.device_status() == 0
