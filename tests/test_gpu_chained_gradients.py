"""The launches inside one public call, and those of a backward pass, may come up while their predecessor drains too: a
training step queued as it is used against the same launches one by one with the device idle in between.  The weight
gradients' reference has no plan launch before it (round-robin tiles), so it cannot repeat a fault of that pair."""

import pytest
import torch

from gated_ffn_ref import assert_within, block
from triton_grouped_gemm_b200 import _lib
from triton_grouped_gemm_b200.ep.autograd import combine_rows, permute_rows
from triton_grouped_gemm_b200.gemm.autograd import grouped_gated_ffn
from triton_grouped_gemm_b200.gemm.BF16.m_grouped_gated_gemm import _m_grouped_gated_grad_launch, _m_grouped_gated_launch
from triton_grouped_gemm_b200.gemm.BF16.m_grouped_gemm_TMA import _m_grouped_gemm_launch

pytestmark = pytest.mark.gpu
DEV = "cuda"

CASES = {
    # tokens, experts, hidden, inter, top_k, rows behind the groups
    "tiny": (3, 4, 64, 40, 2, 1),
    "small": (75, 16, 256, 136, 3, 6),
    "ragged": (700, 9, 520, 264, 4, 3),
    "pairs": (5000, 4, 512, 512, 2, 130),
}


def _problem(case, dtype, seed):
    tokens, experts, hidden, inter, top_k, extra = CASES[case]
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)

    expert = torch.topk(torch.rand(tokens, experts, generator=gen, device=DEV), top_k, dim=1).indices.reshape(-1)
    first = torch.argsort(expert, stable=True)
    pos = torch.empty_like(first)
    pos[first] = torch.arange(first.numel(), device=DEV)
    order = torch.cat([first, first.new_full((extra,), -1)])          # rows that no pair owns
    return dict(x=normal(tokens, hidden), weight=torch.softmax(torch.rand(tokens, top_k, generator=gen, device=DEV), 1), pos=pos,
                order=order, sizes=torch.bincount(expert, minlength=experts), w13=normal(experts, 2 * inter, hidden, std=hidden ** -0.5),
                w2=normal(experts, hidden, inter, std=inter ** -0.5), dout=normal(tokens, hidden), top_k=top_k)


def _step(p):
    """As a user queues it: out and the gradients of x, weight, w13 and w2."""
    x, weight, w13, w2 = (p[n].detach().requires_grad_() for n in ("x", "weight", "w13", "w2"))
    rows = permute_rows(x, p["pos"], p["order"], p["top_k"])
    y = grouped_gated_ffn(rows, w13, w2, p["sizes"])
    out = combine_rows(y, weight, p["pos"], p["order"])
    return (out.detach(),) + torch.autograd.grad(out, (x, weight, w13, w2), p["dout"])


def _weight_gradient(a, b, sizes):
    c = a.new_empty(sizes.numel(), a.shape[1], b.shape[1])
    rc = _lib.load().b200gemm_k_grouped(a.data_ptr(), b.data_ptr(), c.data_ptr(), sizes.data_ptr(), 1, None, None, sizes.numel(),
                                        a.shape[0], a.shape[1], b.shape[1], _lib.dtype_code(a.dtype), None, 0, -1,
                                        _lib.stream_ptr(a.device))
    _lib.check(rc, "b200gemm_k_grouped")
    torch.cuda.synchronize()
    return c


def _one_by_one(p):
    """The same from single launches; also (rows, y, dy, dx of the rows) for the check against 64 bits."""
    sync = torch.cuda.synchronize
    x = p["x"].detach().requires_grad_()
    rows = permute_rows(x, p["pos"], p["order"], p["top_k"])
    sync()
    r, y = rows.detach(), rows.new_empty(rows.shape)
    h, saved, exps = _m_grouped_gated_launch(r, p["w13"], p["sizes"], "silu", save=True, tail=y)
    sync()
    _m_grouped_gemm_launch(h, p["w2"], y, p["sizes"], True)
    sync()
    y.requires_grad_()
    weight = p["weight"].detach().requires_grad_()
    out = combine_rows(y, weight, p["pos"], p["order"])
    sync()
    dy, dweight = torch.autograd.grad(out, (y, weight), p["dout"])
    sync()
    dx_rows = torch.empty_like(dy)
    dgu = _m_grouped_gated_grad_launch(dy, p["w2"], saved, exps, p["sizes"], "silu", tail=dx_rows)
    sync()
    _m_grouped_gemm_launch(dgu, p["w13"], dx_rows, p["sizes"], False)
    sync()
    dw13, dw2 = _weight_gradient(dgu, r, p["sizes"]), _weight_gradient(dy, h, p["sizes"])
    dx, = torch.autograd.grad(rows, x, dx_rows)
    sync()
    return (out.detach(), dx, dweight, dw13, dw2), (r, y.detach(), dy, dx_rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES)
def test_training_step_as_launch_by_launch(case, dtype):
    problems = [_problem(case, dtype, seed) for seed in (1, 2)]       # in turn, so that what is left over differs
    lib = _lib.load()
    pairs = case == "pairs"
    want = []
    for p in problems:
        result, (r, y, dy, dx) = _one_by_one(p)
        n = int(p["sizes"].sum())
        assert not y[n:].any() and not dx[n:].any()
        ref = block(r, p["w13"], p["w2"], p["sizes"].tolist(), "silu", dy)
        for got, name in ((y, "y"), (dx, "dx"), (result[3], "dw13"), (result[4], "dw2")):
            assert_within(got, ref[name], name)
        want.append((result, ref))
    assert lib.b200gemm_set_cta_pair(-1 if pairs else 0) == 0
    try:
        for _ in range(8):
            queued = [_step(p) for p in problems]
            for got, (result, ref) in zip(queued, want):
                for i, (a, b) in enumerate(zip(got, result)):
                    if pairs and i >= 3:                              # another form of the product: within its bounds
                        assert_within(a, ref[("dw13", "dw2")[i - 3]], i)
                    else:
                        assert torch.equal(a, b), i
    finally:
        lib.b200gemm_set_cta_pair(-1)
    assert _lib.device_status() == 0


def test_training_steps_replayed():
    p = _problem("small", torch.bfloat16, 3)
    want = _one_by_one(p)[0]
    lib = _lib.load()
    assert lib.b200gemm_set_cta_pair(0) == 0
    try:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(p)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _step(p)
            again = _step(p)
        for _ in range(4):
            for g in got + again:
                g.zero_()
            graph.replay()
            graph.replay()
            for a, b, c in zip(got, again, want):
                assert torch.equal(a, c) and torch.equal(b, c)
    finally:
        lib.b200gemm_set_cta_pair(-1)
    assert _lib.device_status() == 0
