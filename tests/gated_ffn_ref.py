"""The gated feed-forward block and its gradients in 64 bits, written out, with elementwise bounds on what 16-bit
operands with fp32 accumulation may differ by.

A bound is carried beside every value: a product of 16-bit operands over K terms is off by at most
``acc(K) * sum |a||b|`` (each of K/16 tensor-core steps and the final sum err by at most 2^-22 of the running sum of
magnitudes), a value rounded to 16 bits by eps/2 of itself (and half the smallest denormal), and what a factor is off by
enters a product through the other factor's magnitude."""

import torch

HALF_EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
HALF_TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
# the kept gate and up values, relative to themselves and to their block's maximum: half a mantissa step and half a
# denormal step.  bf16 layers: fp16 with the maximum in [2^14, 2^15): 2^-11 and 2^-25 / 2^14.  fp16 layers: 12 mantissa
# bits, 2^-13, down to 2^-5 of the maximum's power of two, in steps of 2^-17 of it below: 2^-18.
KEPT = {torch.bfloat16: (2.0 ** -11, 2.0 ** -39), torch.float16: (2.0 ** -13, 2.0 ** -18)}


def act_and_slopes(g, act):
    """act(g), act'(g) and an upper bound of |act''|."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s)), 0.5
    c = (2 / torch.pi) ** 0.5
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g), 1.0


def _acc(k):
    return (k / 16 + 2) * 2.0 ** -22


def _round(v, bound, dtype):
    return bound + HALF_EPS[dtype] * (v.abs() + bound) + HALF_TINY[dtype]


def _mm(a, ea, b, eb):
    """a @ b and its bound from the operands' bounds."""
    e = ea @ (b.abs() + eb) + a.abs() @ eb + _acc(a.shape[1]) * ((a.abs() + ea) @ (b.abs() + eb))
    return a @ b, e


def forward_group(x, w13, w2, act, dtype):
    """One expert: dict of (value, bound) for g, u, h (rounded) and y (rounded)."""
    x, w13, w2 = x.double(), w13.double(), w2.double()
    i = w13.shape[0] // 2
    zx, zw = torch.zeros_like(x), torch.zeros_like(w13).t()
    gu, egu = _mm(x, zx, w13.t(), zw)
    g, u, eg, eu = gu[:, :i], gu[:, i:], egu[:, :i], egu[:, i:]
    a, slope, curve = act_and_slopes(g, act)
    ea = (slope.abs() + curve * eg) * eg + 2.0 ** -16 * a.abs()       # __expf's error, at most 2^-17
    h = a * u
    eh = _round(h, ea * (u.abs() + eu) + a.abs() * eu, dtype)
    y, ey = _mm(h, eh, w2.t(), torch.zeros_like(w2).t())
    return dict(x=x, w13=w13, w2=w2, g=(g, eg), u=(u, eu), h=(h, eh), y=(y, _round(y, ey, dtype)))


def backward_group(f, dy, act, dtype):
    """Gradients of one expert: dx, dw13, dw2 as (value, bound)."""
    dy = dy.double()
    zy = torch.zeros_like(dy)
    (g, eg), (u, eu) = f["g"], f["u"]
    rel, floor = KEPT[dtype]

    def kept(v, e):
        m = v.abs() + e
        return e + rel * m + floor * m.amax(1, keepdim=True) if v.shape[0] else e

    eg, eu = kept(g, eg), kept(u, eu)
    a, slope, curve = act_and_slopes(g, act)
    third = 1.0 if act == "silu" else 3.0                             # |act''| moves by less than this per unit
    ea = (slope.abs() + curve * eg) * eg + 2.0 ** -16 * a.abs()
    es = (curve + third * eg) * eg + 2.0 ** -15 * (slope.abs() + a.abs())
    dh, edh = _mm(dy, zy, f["w2"], torch.zeros_like(f["w2"]))
    dg, du = dh * u * slope, dh * a
    edg = edh * (u.abs() + eu) * (slope.abs() + es) + dh.abs() * (eu * (slope.abs() + es) + u.abs() * es) + 2.0 ** -22 * dg.abs()
    edu = edh * (a.abs() + ea) + dh.abs() * ea + 2.0 ** -22 * du.abs()
    dgu = torch.cat((dg, du), 1)
    edgu = torch.cat((_round(dg, edg, dtype), _round(du, edu, dtype)), 1)
    dx, edx = _mm(dgu, edgu, f["w13"], torch.zeros_like(f["w13"]))
    dw13, ew13 = _mm(dgu.t(), edgu.t(), f["x"], torch.zeros_like(f["x"]))
    dw2, ew2 = _mm(dy.t(), zy.t(), f["h"][0], f["h"][1])
    return dict(dx=(dx, _round(dx, edx, dtype)), dw13=(dw13, _round(dw13, ew13, dtype)), dw2=(dw2, _round(dw2, ew2, dtype)))


def block(x, w13, w2, sizes, act, dy=None):
    """The whole block on rows grouped by expert: dict of (value, bound); rows behind the groups are zeros, exactly."""
    dtype, n, m = x.dtype, sum(sizes), x.shape[0]
    parts = [forward_group(xe, w13[e], w2[e], act, dtype) for e, xe in enumerate(x[:n].split(sizes))]

    def rows(name, ps):
        return tuple(torch.cat([p[name][b] for p in ps] + [torch.zeros(m - n, ps[0][name][b].shape[1], dtype=torch.float64,
                                                                       device=x.device)]) for b in range(2))

    out = dict(y=rows("y", parts), h=rows("h", parts))
    if dy is not None:
        grads = [backward_group(p, d, act, dtype) for p, d in zip(parts, dy[:n].split(sizes))]
        out["dx"] = rows("dx", grads)
        for w in ("dw13", "dw2"):
            out[w] = tuple(torch.stack([p[w][b] for p in grads]) for b in range(2))
    return out


def assert_within(got, ref, what):
    value, bound = ref
    off = (got.double() - value).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values out of bounds, worst {float((off / bound).nan_to_num(9e9).max()):.3g} of its bound"
