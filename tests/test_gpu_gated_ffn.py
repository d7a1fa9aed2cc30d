"""The experts' gated feed-forward block against its formulas in 64 bits, elementwise, with derived bounds."""

import pytest
import torch

from gated_ffn_ref import act_and_slopes, assert_within, block
from triton_grouped_gemm_b200 import _lib
from triton_grouped_gemm_b200.gemm.autograd import grouped_gated_ffn
from triton_grouped_gemm_b200.gemm.BF16.m_grouped_gated_gemm import m_grouped_gated_gemm

pytestmark = pytest.mark.gpu
DEV = "cuda"

# sizes, hidden, inter, rows behind the groups
SHAPES = {
    "one_row": ([1], 8, 8, 0),
    "tiny_ragged": ([3, 0, 5], 72, 40, 2),
    "few_rows_each": ([1, 2, 0, 1, 7, 1], 512, 264, 0),
    "tile_edges": ([128, 127, 129, 0, 32, 33], 256, 384, 1),
    "straddling_block": ([130, 0, 257, 64, 1], 200, 1000, 5),
    "wide_tiles": ([1500, 900, 0, 700, 1300, 700, 450, 450], 136, 1032, 3),
    "pair_tiles": ([4100, 0, 3901], 512, 776, 0),
}


def _inputs(sizes, hidden, inter, extra, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    g, m = len(sizes), sum(sizes) + extra

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)

    return (normal(m, hidden), normal(g, 2 * inter, hidden, std=hidden ** -0.5), normal(g, hidden, inter, std=inter ** -0.5),
            normal(m, hidden))


def _run(x, w13, w2, sizes, act, dy):
    x, w13, w2 = (t.detach().requires_grad_() for t in (x, w13, w2))
    y = grouped_gated_ffn(x, w13, w2, torch.tensor(sizes, device=DEV), act)
    return (y.detach(),) + torch.autograd.grad(y, (x, w13, w2), dy)


def _check(got, ref):
    for value, name in zip(got, ("y", "dx", "dw13", "dw2")):
        assert_within(value, ref[name], name)


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_block_and_gradients(shape, dtype, act):
    sizes, hidden, inter, extra = SHAPES[shape]
    x, w13, w2, dy = _inputs(sizes, hidden, inter, extra, dtype)
    ref = block(x, w13, w2, sizes, act, dy)
    got = _run(x, w13, w2, sizes, act, dy)
    assert _lib.device_status() == 0
    _check(got, ref)
    # inference keeps nothing but computes the same bits; the fused product alone is its h
    with torch.no_grad():
        sizes_dev = torch.tensor(sizes, device=DEV, dtype=torch.int32)
        assert torch.equal(grouped_gated_ffn(x, w13, w2, sizes_dev, act), got[0])
        h = m_grouped_gated_gemm(x, w13, sizes_dev, act)
        n = sum(sizes)
        assert_within(h[:n], tuple(t[:n] for t in ref["h"]), "h")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", ["tiny_ragged", "tile_edges", "straddling_block"])
def test_cta_pairs_at_every_size(shape, dtype):
    """The CTA-pair form on shapes the size rule gives to the single-CTA form."""
    sizes, hidden, inter, extra = SHAPES[shape]
    x, w13, w2, dy = _inputs(sizes, hidden, inter, extra, dtype)
    lib = _lib.load()
    assert lib.b200gemm_set_cta_pair(1) == 0
    try:
        got = _run(x, w13, w2, sizes, "silu", dy)
    finally:
        lib.b200gemm_set_cta_pair(-1)
    assert _lib.device_status() == 0
    _check(got, block(x, w13, w2, sizes, "silu", dy))


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -20, 2.0 ** 20])
def test_kept_values_over_the_exponent_range(scale):
    """Gate and up products far from 1, with one column a thousand times larger than its neighbours: the kept values
    are relative to the block's largest, whatever its exponent.  (dh is scaled back so that no gradient overflows.)"""
    sizes, hidden, inter, extra = [40, 3, 129], 64, 96, 0
    x, w13, w2, dy = _inputs(sizes, hidden, inter, extra, torch.bfloat16, seed=3)
    w13 = w13.clone()
    w13[:, inter + 17] *= 1024
    w13[:, inter:] *= scale                                           # u; g stays where silu bends
    w2 = (w2.float() * min(1.0, 1 / scale)).to(torch.bfloat16)
    ref = block(x, w13, w2, sizes, "silu", dy)
    _check(_run(x, w13, w2, sizes, "silu", dy), ref)
    assert _lib.device_status() == 0


def test_gradient_against_differences():
    """<grad, v> against the central difference of the 64-bit block along v: its own error is the third derivative
    times step^2 / 6 (step 1e-4: 1e-8 of the values) and 64-bit cancellation (1e-12); the gradients' bounds cover the rest."""
    sizes, hidden, inter, extra = [37, 0, 90], 72, 56, 0
    x, w13, w2, dy = _inputs(sizes, hidden, inter, extra, torch.bfloat16, seed=5)
    ref = block(x, w13, w2, sizes, "gelu_tanh", dy)
    _, dx, dw13, dw2 = _run(x, w13, w2, sizes, "gelu_tanh", dy)
    gen = torch.Generator(device=DEV).manual_seed(9)
    dirs = [torch.randn(t.shape, generator=gen, device=DEV, dtype=torch.float64) for t in (x, w13, w2)]

    def loss(step):
        total = 0.0
        lo = 0
        for e, s in enumerate(sizes):
            xe, a, b = (t.double() + step * d for t, d in ((x[lo:lo + s], dirs[0][lo:lo + s]), (w13[e], dirs[1][e]), (w2[e], dirs[2][e])))
            gate, up = (xe @ a.t()).chunk(2, 1)
            total = total + ((act_and_slopes(gate, "gelu_tanh")[0] * up) @ b.t() * dy[lo:lo + s].double()).sum()
            lo += s
        return total

    step = 1e-4
    difference = (loss(step) - loss(-step)) / (2 * step)
    inner = sum((g.double() * d).sum() for g, d in zip((dx, dw13, dw2), dirs))
    allowed = sum((ref[n][1] * d.abs()).sum() for n, d in zip(("dx", "dw13", "dw2"), dirs))
    size = sum((g.double() * d).abs().sum() for g, d in zip((dx, dw13, dw2), dirs))
    assert abs(inner - difference) <= allowed + 1e-5 * size
    assert allowed < 0.25 * size                                      # the bound says something


def test_masked_rows_layout():
    g, stride, hidden, inter = 5, 96, 128, 136
    valid = [0, 96, 1, 33, 70]
    x, w13, _, _ = _inputs([stride] * g, hidden, inter, 0, torch.bfloat16, seed=7)
    out = torch.full((g * stride, inter), 7.0, device=DEV, dtype=torch.bfloat16)
    m_grouped_gated_gemm(x, w13, torch.tensor(valid, device=DEV), masked_stride=stride, out=out)
    assert _lib.device_status() == 0
    for e, v in enumerate(valid):
        slot = slice(e * stride, e * stride + v)
        w2 = torch.zeros(hidden, inter, device=DEV, dtype=torch.bfloat16)
        ref = block(x[slot], w13[e:e + 1], w2[None], [v], "silu")["h"]
        assert_within(out[slot], ref, f"slot {e}")
        assert torch.all(out[e * stride + v:(e + 1) * stride] == 7.0)


def test_non_finite_rows_stay_where_they_are():
    """NaN and infinity in one expert's rows and in the rows behind the groups reach no other expert."""
    sizes, hidden, inter, extra = [70, 45, 60], 128, 96, 9
    x, w13, w2, dy = _inputs(sizes, hidden, inter, extra, torch.bfloat16, seed=11)
    clean = _run(x, w13, w2, sizes, "silu", dy)
    x2, dy2 = x.clone(), dy.clone()
    x2[71], x2[80, 3], x2[175:] = float("nan"), float("inf"), float("nan")
    dy2[177] = float("inf")
    y, dx, dw13, dw2 = _run(x2, w13, w2, sizes, "silu", dy2)
    keep = torch.ones(sum(sizes) + extra, dtype=torch.bool, device=DEV)
    keep[[71, 80]] = False
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
    for e in (0, 2):
        assert torch.equal(dw13[e], clean[2][e]) and torch.equal(dw2[e], clean[3][e])
    assert y[71].isnan().all() and dx[71].isnan().all()
    assert dx[80].isnan().any() and dw13[1].isnan().any()
    assert _lib.device_status() == 0


def test_group_sizes_past_the_rows_are_cut_off_and_flagged():
    sizes, hidden, inter, _ = [40, 30, 20], 64, 64, 0
    x, w13, w2, dy = _inputs(sizes, hidden, inter, 0, torch.bfloat16, seed=13)
    good = _run(x, w13, w2, sizes, "silu", dy)
    assert _lib.device_status() == 0
    got = _run(x, w13, w2, [40, 30, 4000], "silu", dy)
    assert _lib.device_status() == 0x10
    for a, b in zip(got[:2], good[:2]):
        assert torch.equal(a, b)


def test_no_rows_and_no_groups():
    w13 = torch.randn(2, 32, 16, device=DEV).bfloat16().requires_grad_()
    w2 = torch.randn(2, 16, 16, device=DEV).bfloat16().requires_grad_()
    x = torch.zeros(0, 16, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = grouped_gated_ffn(x, w13, w2, torch.zeros(2, dtype=torch.int64, device=DEV))
    dx, dw13, dw2 = torch.autograd.grad(y, (x, w13, w2), torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 16) and not dw13.any() and not dw2.any()
    x = torch.randn(5, 16, device=DEV).bfloat16().requires_grad_()
    y = grouped_gated_ffn(x, w13, w2, torch.zeros(2, dtype=torch.int64, device=DEV))
    dx, dw13 = torch.autograd.grad(y, (x, w13), torch.ones_like(y))
    assert not y.any() and not dx.any() and not dw13.any()
    y = grouped_gated_ffn(x, w13[:0], w2[:0], torch.zeros(0, dtype=torch.int64, device=DEV))
    assert not y.any() and not torch.autograd.grad(y, x, torch.ones_like(y))[0].any()


def test_single_gradients_strides_and_offsets():
    """Every subset of wanted gradients gives the same bits; operands and gradients that are views are taken too."""
    sizes, hidden, inter, extra = [40, 0, 33], 64, 48, 2
    x, w13, w2, dy = _inputs(sizes, hidden, inter, extra, torch.bfloat16, seed=17)
    full = _run(x, w13, w2, sizes, "silu", dy)[1:]
    s = torch.tensor(sizes, device=DEV)
    for which in range(3):
        leaves = [t.detach().requires_grad_(i == which) for i, t in enumerate((x, w13, w2))]
        y = grouped_gated_ffn(*leaves, s)
        assert torch.equal(torch.autograd.grad(y, leaves[which], dy)[0], full[which])
    xt = x.t().contiguous().t().requires_grad_()                      # column-major view
    w13t = w13.transpose(1, 2).contiguous().transpose(1, 2).requires_grad_()
    y = grouped_gated_ffn(xt, w13t, w2, s)
    odd = torch.empty(dy.numel() + 1, device=DEV, dtype=dy.dtype)[1:].view_as(dy).copy_(dy)   # 2 bytes off 16
    got = torch.autograd.grad(y, (xt, w13t), odd)
    assert torch.equal(got[0], full[0]) and torch.equal(got[1], full[1])
    y = grouped_gated_ffn(xt, w13t, w2, s)
    y.sum().backward()                                                # a gradient with strides of zero
    ones = _run(x, w13, w2, sizes, "silu", torch.ones_like(dy))
    assert torch.equal(xt.grad, ones[1]) and torch.equal(w13t.grad, ones[2])


def test_broadcast_inputs_sum_their_gradients():
    """One token's row in every row of x, one expert's weights in every expert: the gradients of the shared tensors are
    the sums over the copies (of 16-bit gradients, which autograd adds up)."""
    sizes, hidden, inter = [20, 0, 45], 64, 48
    x1, w13, w2, _ = _inputs([1, 0, 0], hidden, inter, 0, torch.bfloat16, seed=37)
    dy = _inputs(sizes, hidden, inter, 0, torch.bfloat16, seed=38)[3]
    s = torch.tensor(sizes, device=DEV)
    leaves = [t.detach().clone().requires_grad_() for t in (x1, w13[:1], w2[:1])]
    y = grouped_gated_ffn(leaves[0].expand(65, -1), leaves[1].expand(3, -1, -1), leaves[2].expand(3, -1, -1), s)
    got = torch.autograd.grad(y, leaves, dy)
    full = _run(x1.expand(65, -1).contiguous(), w13[:1].expand(3, -1, -1).contiguous(), w2[:1].expand(3, -1, -1).contiguous(),
                sizes, "silu", dy)[1:]
    for a, b in zip(got, full):
        want = b.double().sum(0, keepdim=True)
        assert ((a.double() - want).abs() <= 2.0 ** -8 * b.double().abs().sum(0, keepdim=True)).all()


def test_two_threads_at_once():
    """Calls from several host threads, each on its own stream."""
    import threading

    cases = [(_inputs(sz, 128, 96, 1, torch.bfloat16, seed=i), sz) for i, sz in enumerate(([40, 0, 9], [1, 2, 3], [0, 0, 70], [33, 33, 33]))]
    want = [_run(x, w13, w2, sz, "silu", dy) for (x, w13, w2, dy), sz in cases]
    torch.cuda.synchronize()
    got = [None] * len(cases)

    def work(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(5):
                (x, w13, w2, dy), sz = cases[i]
                got[i] = _run(x, w13, w2, sz, "silu", dy)
        st.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert _lib.device_status() == 0


def test_fewer_sms():
    sizes, hidden, inter, extra = SHAPES["straddling_block"]
    x, w13, _, _ = _inputs(sizes, hidden, inter, extra, torch.bfloat16, seed=41)
    s = torch.tensor(sizes, device=DEV)
    n = sum(sizes)
    assert torch.equal(m_grouped_gated_gemm(x, w13, s, numSM=3)[:n], m_grouped_gated_gemm(x, w13, s)[:n])


def test_repeatable_and_on_other_streams():
    sizes, hidden, inter, extra = SHAPES["straddling_block"]
    x, w13, w2, dy = _inputs(sizes, hidden, inter, extra, torch.bfloat16, seed=19)
    first = _run(x, w13, w2, sizes, "silu", dy)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            results.append(_run(x, w13, w2, sizes, "silu", dy))
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, first))


def test_captured_forward_and_backward_replay():
    sizes, hidden, inter, extra = [50, 0, 70, 9], 128, 96, 4
    x, w13, w2, dy = _inputs(sizes, hidden, inter, extra, torch.bfloat16, seed=23)
    sx, sdy, ss = x.clone(), dy.clone(), torch.tensor(sizes, device=DEV)

    def step():
        a, b, c = sx.detach().requires_grad_(), w13.detach().requires_grad_(), w2.detach().requires_grad_()
        y = grouped_gated_ffn(a, b, c, ss)
        return (y.detach(),) + torch.autograd.grad(y, (a, b, c), sdy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed, new_sizes in ((29, [129, 0, 4, 0]), (31, [1, 1, 1, 100])):
        x2, _, _, dy2 = _inputs(sizes, hidden, inter, extra, torch.bfloat16, seed=seed)
        sx.copy_(x2)
        sdy.copy_(dy2)
        ss.copy_(torch.tensor(new_sizes, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        eager = _run(x2, w13, w2, new_sizes, "silu", dy2)
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_full_and_partial_tiles_in_turn(dtype):
    """Every block of the launch gets a full tile, then a group's last one whose rows end inside one of its warps, then a
    full one again: what a warp stages for the third may not overtake the first one's store."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    sizes = ([128 * sms] + [(20, 52, 84, 116)[i % 4] for i in range(sms)]) * 3
    x, w13, w2, dy = _inputs(sizes, 16, 64, 0, dtype)
    want = _run(x, w13, w2, sizes, "silu", dy)
    _check(want, block(x, w13, w2, sizes, "silu", dy))
    group_sizes = torch.tensor(sizes, device=DEV)
    for _ in range(30):
        with torch.no_grad():
            assert torch.equal(grouped_gated_ffn(x, w13, w2, group_sizes), want[0])
        for value, first in zip(_run(x, w13, w2, sizes, "silu", dy), want):
            assert torch.equal(value, first)
