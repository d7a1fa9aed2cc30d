"""4-bit weight products and their quantiser against their definitions in 64 bits.

Tolerance of a product, elementwise: values of `a` times whole numbers are exact in fp32; a group's sum and the sum over
the groups err by at most 2^-22 per tensor-core step and addition of the running sum of magnitudes; one rounding of
eps/2 at the end (and half the smallest denormal of fp16)."""

import pytest
import torch

from gated_ffn_ref import HALF_EPS, HALF_TINY, act_and_slopes, assert_within
from triton_grouped_gemm_b200 import _lib
from triton_grouped_gemm_b200.gemm.W4.m_grouped_gemm_w4 import m_grouped_gemm_w4, m_grouped_gemm_w4_gated
from triton_grouped_gemm_b200.quant.per_group_cast import per_group_cast_to_w4

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _weights(g, rows, k, gs, zero, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randint(0, 256, (g, rows, k // 2), generator=gen, device=DEV, dtype=torch.uint8)
    scale = (torch.rand(g, rows, k // gs, generator=gen, device=DEV) * 0.1 + 0.01).to(dtype)
    z = torch.randint(0, 16, (g, rows, k // gs), generator=gen, device=DEV, dtype=torch.uint8) if zero else None
    return q, scale, z


def _values(b):
    q, scale, z = b
    gs = 2 * q.shape[-1] // scale.shape[-1]
    whole = torch.stack((q & 15, q >> 4), -1).flatten(-2).double()
    z = 8.0 if z is None else z.double().repeat_interleave(gs, -1)
    return (whole - z) * scale.double().repeat_interleave(gs, -1)


def _activations(m, k, dtype, seed=1):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(m, k, generator=gen, device=DEV).to(dtype)


def _reference(a, b, sizes, act=None):
    w = _values(b)
    values, bounds, lo = [], [], 0
    for e, s in enumerate(sizes):
        x = a[lo:lo + s].double()
        c = x @ w[e].t()
        ec = (a.shape[1] / 16 + 16) * 2.0 ** -22 * (x.abs() @ w[e].abs().t())
        if act:
            (g, u), (eg, eu) = c.chunk(2, 1), ec.chunk(2, 1)
            v, slope, curve = act_and_slopes(g, act)
            ev = (slope.abs() + curve * eg) * eg + 2.0 ** -16 * v.abs()
            c, ec = v * u, ev * (u.abs() + eu) + v.abs() * eu
        values.append(c)
        bounds.append(ec + HALF_EPS[a.dtype] * (c.abs() + ec) + HALF_TINY[a.dtype])
        lo += s
    return torch.cat(values), torch.cat(bounds)


CASES = [
    # sizes, rows of weights (even), k, group size
    ([1], 2, 32, 32),
    ([1, 0, 2, 0, 0, 5], 72, 64, 64),
    ([0, 0, 8], 64, 768, 128),
    ([1, 1, 1, 1, 1, 1, 1, 1], 96, 2048, 128),
    ([9, 0, 33, 1], 130, 288, 32),
    ([7, 32, 64, 0, 31], 250, 1088, 64),
    ([2, 100], 10, 4352, 32),            # scales of more than one window
    ([3, 3], 34, 8320, 64),
    ([40, 3], 6, 17024, 128),
]


@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_products(case, dtype, zero):
    sizes, rows, k, gs = CASES[case]
    b = _weights(len(sizes), rows, k, gs, zero, dtype, seed=case)
    m = sum(sizes)
    a = _activations(m + 2, k, dtype, seed=case + 100)
    out = torch.full((m + 2, rows), 3.0, device=DEV, dtype=dtype)
    got = m_grouped_gemm_w4(a, b, torch.tensor(sizes, device=DEV), out=out)
    assert got is out
    assert_within(out[:m], _reference(a, b, sizes), "product")
    assert torch.all(out[m:] == 3.0)                                  # rows behind the groups
    half = a * torch.tensor(0.25, device=DEV, dtype=dtype)            # keeps fp16 products in range
    for act in ("silu", "gelu_tanh"):
        got = m_grouped_gemm_w4_gated(half, b, torch.tensor(sizes, device=DEV, dtype=torch.int32), act)
        assert_within(got[:m], _reference(half, b, sizes, act), act)
    assert _lib.device_status() == 0


def test_many_experts_few_rows():
    g, rows, k, gs = 1024, 34, 64, 32
    gen = torch.Generator().manual_seed(5)
    sizes = (torch.rand(g, generator=gen) < 0.1).long() * torch.randint(1, 4, (g,), generator=gen)
    b = _weights(g, rows, k, gs, True, torch.bfloat16)
    a = _activations(int(sizes.sum()), k, torch.bfloat16)
    got = m_grouped_gemm_w4(a, b, sizes.to(DEV))
    assert_within(got, _reference(a, b, sizes.tolist()), "1024 experts")


def test_rows_do_not_depend_on_their_neighbours():
    """A row gives the same bits alone and in company, in whichever form of the kernel its batch runs, up to the order
    of the partial sums, which the two forms split differently: within the bound."""
    rows, k, gs = 130, 1024, 64
    b = _weights(3, rows, k, gs, True, torch.float16)
    a = _activations(45, k, torch.float16)
    sizes = [20, 5, 20]
    ref = _reference(a, b, sizes)
    both = m_grouped_gemm_w4(a, b, torch.tensor(sizes, device=DEV))
    assert_within(both, ref, "together")
    again = m_grouped_gemm_w4(a, b, torch.tensor(sizes, device=DEV))
    assert torch.equal(both, again)
    alone = m_grouped_gemm_w4(a[20:25].contiguous(), b, torch.tensor([0, 5, 0], device=DEV))
    assert_within(alone, tuple(t[20:25] for t in ref), "alone")


def test_non_finite_rows_stay_where_they_are():
    b = _weights(2, 66, 256, 32, False, torch.bfloat16)
    a = _activations(12, 256, torch.bfloat16)
    s = torch.tensor([9, 3], device=DEV)
    clean = m_grouped_gemm_w4(a, b, s)
    a2 = a.clone()
    a2[4], a2[10, 7] = float("nan"), float("inf")
    got = m_grouped_gemm_w4(a2, b, s)
    keep = [r for r in range(12) if r not in (4, 10)]
    assert torch.equal(got[keep], clean[keep]) and got[4].isnan().all() and not got[10].isfinite().all()


def test_group_sizes_past_the_rows_are_cut_off_and_flagged():
    b = _weights(3, 40, 128, 64, False, torch.bfloat16)
    a = _activations(6, 128, torch.bfloat16)
    good = m_grouped_gemm_w4(a, b, torch.tensor([2, 3, 1], device=DEV))
    assert _lib.device_status() == 0
    for bad in ([2, 3, 9], [2, 3, 2 ** 31], [2, 3, 2 ** 62]):
        got = m_grouped_gemm_w4(a, b, torch.tensor(bad, device=DEV))
        assert _lib.device_status() == 0x10 and torch.equal(got, good)
    got = m_grouped_gemm_w4(a, b, torch.tensor([2, 2 ** 40, 1], device=DEV))     # the second takes all that is left
    assert _lib.device_status() == 0x10 and torch.equal(got[:2], good[:2])
    got = m_grouped_gemm_w4(a, b, torch.tensor([-5, 3, 3], device=DEV))
    assert _lib.device_status() == 0
    assert torch.equal(got, m_grouped_gemm_w4(a, b, torch.tensor([0, 3, 3], device=DEV)))


def test_no_rows():
    b = _weights(3, 40, 128, 64, False, torch.bfloat16)
    out = m_grouped_gemm_w4(_activations(0, 128, torch.bfloat16), b, torch.zeros(3, dtype=torch.int64, device=DEV))
    assert out.shape == (0, 40)
    out = torch.full((4, 40), 5.0, device=DEV, dtype=torch.bfloat16)
    m_grouped_gemm_w4(_activations(4, 128, torch.bfloat16), b, torch.zeros(3, dtype=torch.int64, device=DEV), out=out)
    assert torch.all(out == 5.0) and _lib.device_status() == 0


def test_fewer_sms_and_concurrent_streams():
    b = _weights(6, 200, 512, 64, True, torch.bfloat16)
    sizes = torch.tensor([3, 0, 20, 1, 0, 9], device=DEV)
    a = _activations(33, 512, torch.bfloat16)
    want = m_grouped_gemm_w4(a, b, sizes)
    assert torch.equal(m_grouped_gemm_w4(a, b, sizes, num_sms=2), want)
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            got += [m_grouped_gemm_w4(a, b, sizes) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got) and _lib.device_status() == 0


def test_scales_off_every_alignment():
    """Scales and zeros that begin 2 and 1 bytes off 16, an odd number of groups per row."""
    g, rows, k, gs = 2, 50, 96, 32
    q, scale, z = _weights(g, rows, k, gs, True, torch.bfloat16)
    s_off = torch.empty(scale.numel() + 1, device=DEV, dtype=scale.dtype)[1:].view_as(scale).copy_(scale)
    z_off = torch.empty(z.numel() + 1, device=DEV, dtype=z.dtype)[1:].view_as(z).copy_(z)
    a = _activations(5, k, torch.bfloat16)
    s = torch.tensor([1, 4], device=DEV)
    got = m_grouped_gemm_w4(a, (q, s_off, z_off), s)
    assert_within(got, _reference(a, (q, scale, z), [1, 4]), "offset scales")


def test_captured_call_replays_on_new_sizes():
    b = _weights(4, 70, 512, 128, True, torch.bfloat16)
    a = _activations(20, 512, torch.bfloat16)
    s = torch.tensor([5, 5, 5, 5], device=DEV)
    m_grouped_gemm_w4_gated(a, b, s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m_grouped_gemm_w4_gated(a, b, s)
    for sizes in ([20, 0, 0, 0], [1, 0, 18, 1]):
        s.copy_(torch.tensor(sizes, device=DEV))
        a.copy_(_activations(20, 512, torch.bfloat16, seed=sum(sizes[:2]) + 7))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, m_grouped_gemm_w4_gated(a, b, torch.tensor(sizes, device=DEV)))


# ------------------------------------------------------------------------------------------- quantiser
def _quant_reference(w, gs, symmetric):
    """The definition in fp32 on the host (every operation of it is one correctly rounded fp32 operation)."""
    v = w.cpu().float().unflatten(-1, (-1, gs))
    lo, hi = v.amin(-1).clamp(max=0), v.amax(-1).clamp(min=0)
    exact = torch.maximum(hi, -lo) / 7 if symmetric else (hi - lo) / 15
    scale = exact.to(w.dtype)
    s = scale.float()
    live = s > 0
    z = torch.full_like(s, 8.0) if symmetric else torch.where(live, torch.round(-lo / s).clamp(0, 15), torch.zeros_like(s))
    q = torch.where(live.unsqueeze(-1), torch.round(v / s.unsqueeze(-1)), torch.zeros_like(v)) + z.unsqueeze(-1)
    q = q.clamp(0, 15).to(torch.uint8).flatten(-2)
    return q[..., ::2] | (q[..., 1::2] << 4), scale, None if symmetric else z.to(torch.uint8)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gs", [32, 64, 128])
def test_quantiser_bytes_scales_and_zeros(gs, dtype, symmetric):
    gen = torch.Generator().manual_seed(gs)
    w = (torch.randn(3, 37, 5 * gs, generator=gen) * torch.rand(3, 37, 1, generator=gen).mul(8).exp2() * 2.0 ** -8).to(dtype)
    w[0, 0] = 0                                                       # a row of zeros
    w[0, 1] = w[0, 1].abs()                                           # one sign only
    w[0, 2] = -w[0, 2].abs()
    w[0, 3] = torch.finfo(dtype).smallest_normal                      # scales that round to zero or to a denormal
    w[0, 4] = torch.finfo(dtype).max * (1 - 2.0 ** -6)
    if not symmetric:
        w[0, 4] = w[0, 4] / 2
    q, s, z = per_group_cast_to_w4(w.to(DEV), gs, symmetric)
    rq, rs, rz = _quant_reference(w, gs, symmetric)
    assert torch.equal(q.cpu(), rq) and torch.equal(s.cpu(), rs)
    assert (z is None) if symmetric else torch.equal(z.cpu(), rz)


def test_quantised_weights_are_near():
    """Asymmetric: off by at most half a step plus what rounding the scale (15 steps of eps/2) and the zero (half a step)
    may add at the ends; symmetric: half a step, plus 7 steps of eps/2."""
    w = torch.randn(2, 64, 512, device=DEV).to(torch.bfloat16)
    for symmetric, steps in ((True, 0.5 + 8 * 2.0 ** -8), (False, 1.0 + 15 * 2.0 ** -8)):
        b = per_group_cast_to_w4(w, 64, symmetric)
        off = (_values(b) - w.double()).abs() / b[1].double().repeat_interleave(64, -1)
        assert off.max() <= steps
