"""Group sizes that name more rows than there are: every product of a group works on the rows that exist, the status word
says so, and no size, however large, stretches a kernel's loop (the cut itself is tested on the host)."""

import pytest
import torch

from triton_grouped_gemm_b200 import _lib
from triton_grouped_gemm_b200.gemm.autograd import grouped_gated_ffn
from triton_grouped_gemm_b200.gemm.BF16.k_grouped_gemm_TMA import k_grouped_gemm
from triton_grouped_gemm_b200.gemm.FP8.k_grouped_gemm_block_scaled import k_grouped_fp8_block_scaled
from triton_grouped_gemm_b200.gemm.FP8.k_grouped_gemm_channel_expert import matmul as k_grouped_fp8_rowcol

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOO_LARGE = [21, 4000, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 20, 2 ** 62]


def _normal(*shape, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=gen, device=DEV).bfloat16()


@pytest.mark.parametrize("last", TOO_LARGE)
def test_gated_block_gives_the_gradients_of_the_cut_sizes(last):
    x, w13, w2, dy = _normal(90, 64), _normal(4, 128, 64, seed=1), _normal(4, 64, 64, seed=2), _normal(90, 64, seed=3)

    def run(sizes):
        leaves = [t.detach().requires_grad_() for t in (x, w13, w2)]
        y = grouped_gated_ffn(*leaves, torch.tensor(sizes, device=DEV))
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    good = run([40, 30, 20, 0])
    assert _lib.device_status() == 0
    got = run([40, 30, last, 7])
    assert _lib.device_status() == 0x10
    for a, b in zip(got, good):
        assert torch.equal(a, b)


@pytest.mark.parametrize("pair", [0, 1])
@pytest.mark.parametrize("last", TOO_LARGE)
def test_k_grouped(last, pair):
    a, b = _normal(90, 256), _normal(90, 264, seed=1)
    lib = _lib.load()
    assert lib.b200gemm_set_cta_pair(pair) == 0
    try:
        good = k_grouped_gemm(a, b, torch.tensor([40, -3, 30, 20, 0], device=DEV))
        assert _lib.device_status() == 0
        sizes = torch.tensor([40, -3, 30, last, last], device=DEV)
        got = k_grouped_gemm(a, b, sizes)
        assert _lib.device_status() == 0x10 and torch.equal(got, good)
        if last < 2 ** 31:
            assert torch.equal(k_grouped_gemm(a, b, sizes.int()), good) and _lib.device_status() == 0x10
            starts = torch.tensor([0, 40, 40, 70, 90], device=DEV)
            ends = torch.tensor([40, 0, 70, 70 + last if last < 2 ** 30 else last, last], device=DEV)
            assert torch.equal(k_grouped_gemm(a, b, sizes, starts, ends), good) and _lib.device_status() == 0x10
    finally:
        lib.b200gemm_set_cta_pair(-1)


@pytest.mark.parametrize("last", TOO_LARGE)
def test_k_grouped_without_a_plan(last):
    a, b = _normal(90, 64), _normal(90, 72, seed=1)
    lib = _lib.load()

    def run(sizes):
        c = torch.empty(len(sizes), 64, 72, device=DEV, dtype=torch.bfloat16)
        s = torch.tensor(sizes, device=DEV)
        rc = lib.b200gemm_k_grouped(a.data_ptr(), b.data_ptr(), c.data_ptr(), s.data_ptr(), 1, None, None, len(sizes), 90, 64, 72,
                                    0, None, 0, -1, _lib.stream_ptr(a.device))
        _lib.check(rc, "b200gemm_k_grouped")
        return c

    good = run([40, 30, 20, 0])
    assert _lib.device_status() == 0
    got = run([40, 30, last, 9])
    assert _lib.device_status() == 0x10 and torch.equal(got, good)


@pytest.mark.parametrize("last", [256, 2 ** 31 - 128, 2 ** 31, 2 ** 32 + 128, 2 ** 62])
def test_k_grouped_fp8(last):
    """Sizes are multiples of 128 here, the unit of both layouts."""
    x8, y8 = (_normal(256, 512, seed=s).to(torch.float8_e4m3fn) for s in (0, 1))
    good_sizes, bad_sizes = (torch.tensor(s, device=DEV) for s in ([128, 256, 128, 0], [128, 256, last, 128]))
    scale = torch.rand(4, 256, device=DEV).t()
    blocks = torch.rand(2, 4, device=DEV)
    for call in (lambda s: k_grouped_fp8_rowcol(x8, scale, y8, scale, s, 256, 256, 512, 4),
                 lambda s: k_grouped_fp8_block_scaled((x8, blocks), (y8, blocks), s)):
        good = call(good_sizes)
        assert _lib.device_status() == 0
        assert torch.equal(call(bad_sizes), good) and _lib.device_status() == 0x10
