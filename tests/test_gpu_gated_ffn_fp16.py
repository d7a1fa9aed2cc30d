"""What fp16 layers keep of the gate and up products for their gradients: values far below their block's largest, and
values that are not finite."""

import pytest
import torch

import gated_ffn_ref
from gated_ffn_ref import block
from test_gpu_gated_ffn import DEV, _check, _inputs, _run
from triton_grouped_gemm_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("half", ["gate", "up"])
@pytest.mark.parametrize("scale,outlier", [(2.0 ** -9, 1024), (1.0, 1024), (1.0, 4), (64.0, 64)])
def test_columns_beside_a_much_larger_one_lose_no_more_than_fp16_would(scale, outlier, half, monkeypatch):
    """One column is `outlier` times its neighbours.  The bounds take a kept value to be off by fp16's 2^-11 of itself, as if
    each had a 16-bit number of its own, and by 2^-23 of the row's largest where it is below 2^-12 of that.  Experts with one
    row: an element of dW13 is then a single product, so no sum over rows hides what a column has lost."""
    monkeypatch.setitem(gated_ffn_ref.KEPT, torch.float16, (2.0 ** -11, 2.0 ** -23))
    sizes, hidden, inter = [1] * 24 + [0, 40, 129], 64, 96
    x, w13, w2, dy = _inputs(sizes, hidden, inter, 0, torch.float16, seed=3)
    w13 = w13.clone()
    first = 0 if half == "gate" else inter
    w13[:, first + 17] *= outlier
    w13[:, first:first + inter] *= scale
    w2 = (w2.float() * min(1.0, 1 / scale)).half()
    dy = (dy.float() * (1 / outlier if half == "gate" else 1.0)).half()    # keeps h's column and the sums over it in range
    _check(_run(x, w13, w2, sizes, "silu", dy), block(x, w13, w2, sizes, "silu", dy))
    assert _lib.device_status() == 0


def test_rows_of_the_weight_gradient_against_fp16_gate_and_up():
    """dW13 row by row, with one up column a thousand times the others: its error in 2-norm against that of the same
    gradient from gate and up products rounded to fp16.  Both differ from the exact one by rounding errors of at most 2^-11
    of each kept value and by the same rounding of dg, du and dW13, so neither can be more than twice the other in every
    term; sums of such terms over 200 rows and 128 columns stay within that factor."""
    sizes, hidden, inter = [70, 130], 128, 64
    x, w13, w2, dy = _inputs(sizes, hidden, inter, 0, torch.float16, seed=5)
    w13 = w13.clone()
    w13[:, inter + 17] *= 1024
    got = _run(x, w13, w2, sizes, "silu", dy)[2].double()
    lo = 0
    for e, s in enumerate(sizes):
        xe, de = x[lo:lo + s].double(), dy[lo:lo + s].double()
        gu = xe @ w13[e].double().t()

        def gradient(gate_up, rounded):
            gate, up = gate_up.chunk(2, 1)
            sig = torch.sigmoid(gate)
            dh = de @ w2[e].double()
            dgu = torch.cat((dh * up * sig * (1 + gate * (1 - sig)), dh * gate * sig), 1)
            if rounded:
                dgu = dgu.half().double()
            dw = dgu.t() @ xe
            return dw.half().double() if rounded else dw

        exact = gradient(gu, False)
        base = (gradient(gu.half().double(), True) - exact).norm(dim=1)
        assert ((got[e] - exact).norm(dim=1) <= 2 * base).all()
        lo += s


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_non_finite_rows_stay_where_they_are(act):
    """NaN and infinity in one expert's rows and in the rows behind the groups reach no other expert, and no other row."""
    sizes, hidden, inter, extra = [70, 45, 60], 128, 96, 9
    x, w13, w2, dy = _inputs(sizes, hidden, inter, extra, torch.float16, seed=11)
    clean = _run(x, w13, w2, sizes, act, dy)
    x2, dy2 = x.clone(), dy.clone()
    x2[71], x2[80, 3], x2[175:] = float("nan"), float("inf"), float("nan")
    dy2[177] = float("inf")
    y, dx, dw13, dw2 = _run(x2, w13, w2, sizes, act, dy2)
    keep = torch.ones(sum(sizes) + extra, dtype=torch.bool, device=DEV)
    keep[[71, 80]] = False
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
    for e in (0, 2):
        assert torch.equal(dw13[e], clean[2][e]) and torch.equal(dw2[e], clean[3][e])
    assert y[71].isnan().all() and dx[71].isnan().all()
    assert dx[80].isnan().any() and dw13[1].isnan().any()
    assert _lib.device_status() == 0
