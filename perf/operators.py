"""Operators around the experts' grouped products of a mixture-of-experts layer, each in its plain form
and as the call a user of this package makes:

  gated_ffn   the experts' gated feed-forward block y = (act(x Wg^T) * (x Wu^T)) W2^T on grouped rows, forward
              alone (serving) or with the gradients of x and of both weight tensors (training)
  w4          M-grouped products with 4-bit weights and group scales for few rows per expert (decoding), plain
              and as the gated gate+up projection
  permute     a token's row to the rows of its top-k experts, with the gradient of the tokens
  combine     the router-weighted sum of a token's expert rows, with the gradients of the rows and of the weights

`own` selects the package's operators; otherwise the same values come from elementary torch operations in 32 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # ---- the feed-forward block of 128 experts of hidden size 2048 and intermediate size 768
        # a decoding step of 16 sequences, top-8: one row or two for most experts; the weights' bytes count
        _ffn("ffn_decode", rows=128, groups=128, active=80, hidden=2048, inter=768, dtype="bf16", act="silu", train=False),
        # a prefill batch
        _ffn("ffn_prefill", rows=32768, groups=128, active=128, hidden=2048, inter=768, dtype="bf16", act="silu", train=False),
        # a training step of the benchmark's size: 81 920 tokens, top-8
        _ffn("ffn_train", rows=655360, groups=128, active=128, hidden=2048, inter=768, dtype="bf16", act="silu", train=True),
        # a fine-tuning step of a small layer in fp16: sizes off every tile border, experts without rows
        _ffn("ffn_train_ragged", rows=5003, groups=16, active=13, hidden=1032, inter=1000, dtype="fp16", act="gelu_tanh",
             train=True),
        # ---- 4-bit weights
        # one sequence: the eight experts of one token, gate+up
        _w4("w4_gated_token", rows=8, groups=128, active=8, n=768, k=2048, group_size=128, zero=False, dtype="bf16", gated=True),
        # the same step's down projection
        _w4("w4_down_token", rows=8, groups=128, active=8, n=2048, k=768, group_size=64, zero=True, dtype="bf16", gated=False),
        # 32 sequences of a layer of hidden size 4096: nearly every expert has a row
        _w4("w4_gated_batch", rows=256, groups=128, active=112, n=1024, k=4096, group_size=128, zero=True, dtype="fp16",
            gated=True),
        # few experts, many rows each, small groups, an output width off every tile border
        _w4("w4_wide", rows=250, groups=8, active=7, n=5003, k=4096, group_size=32, zero=False, dtype="bf16", gated=False),
        # ---- rows between tokens and experts
        # a training step of the benchmark's size, both directions
        _rows("permute_train", "permute", tokens=81920, top_k=8, hidden=2048, dtype="bf16"),
        _rows("combine_train", "combine", tokens=81920, top_k=8, hidden=2048, dtype="bf16"),
        # a short sequence of a small layer, top-2
        _rows("permute_small", "permute", tokens=333, top_k=2, hidden=1032, dtype="fp16"),
        _rows("combine_small", "combine", tokens=333, top_k=2, hidden=1032, dtype="fp16"),
    ]


def _ffn(name, rows, groups, active, hidden, inter, dtype, act, train):
    c = dict(op="gated_ffn", rows=rows, groups=groups, active=active, hidden=hidden, inter=inter, dtype=dtype, act=act, train=train)
    return dict(c, name=name) if name else c


def _w4(name, rows, groups, active, n, k, group_size, zero, dtype, gated):
    c = dict(op="w4", rows=rows, groups=groups, active=active, n=n, k=k, group_size=group_size, zero=zero, dtype=dtype, gated=gated)
    return dict(c, name=name) if name else c


def _rows(name, op, tokens, top_k, hidden, dtype):
    c = dict(op=op, tokens=tokens, top_k=top_k, hidden=hidden, dtype=dtype)
    return dict(c, name=name) if name else c


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("gated_ffn", "w4", "permute", "combine"))
    dtype = rng.choice(("bf16", "fp16"))
    if op == "gated_ffn":
        # rows from one to a long prefill; widths are multiples of 8 (16-byte rows)
        while True:
            groups = _spread(rng, 1, 128)
            rows = _spread(rng, 1, 200000)
            hidden, inter = 8 * _spread(rng, 8, 512), 8 * _spread(rng, 4, 256)
            active = min(rows, rng.randint(max(1, groups // 2), groups))
            c = _ffn("", rows, groups, active, hidden, inter, dtype, rng.choice(("silu", "gelu_tanh")), rng.random() < 0.6)
            w = work(c)
            if w["flops"] <= 8e12 and w["bytes"] <= 1e10:
                return c
    if op == "w4":
        group_size = rng.choice((32, 64, 128))
        groups, rows = _spread(rng, 4, 128), _spread(rng, 1, 256)
        active = min(rows, rng.randint(max(1, groups // 4), groups))
        return _w4("", rows, groups, active, _spread(rng, 40, 5003), group_size * _spread(rng, 2, 4096 // group_size),
                   group_size, rng.random() < 0.5, dtype, rng.random() < 0.5)
    top_k, hidden = rng.randint(1, 8), 8 * _spread(rng, 8, 512)
    tokens = _spread(rng, 1, min(81920, 81920 * 8 * 2048 // (top_k * hidden)))
    return _rows("", op, tokens, top_k, hidden, dtype)


def work(case):
    if case["op"] == "gated_ffn":
        m, h, i, g, a = (case[k] for k in ("rows", "hidden", "inter", "groups", "active"))
        fwd = 2 * (m * h + a * 3 * i * h + m * h)                            # x, the weights of experts with rows, y
        if not case["train"]:
            return {"bytes": fwd, "flops": 6.0 * m * i * h}
        return {"bytes": fwd + 2 * (m * h + m * h + g * 3 * i * h), "flops": 18.0 * m * i * h}   # dy, dx, dW13 and dW2
    if case["op"] == "w4":
        r, a, n, k, gs = (case[x] for x in ("rows", "active", "n", "k", "group_size"))
        wn = 2 * n if case["gated"] else n
        per_row = k / 2 + (k // gs) * (3 if case["zero"] else 2)
        return {"bytes": a * wn * per_row + 2 * r * (k + n), "flops": 2.0 * r * wn * k}
    t, kk, h = case["tokens"], case["top_k"], case["hidden"]
    if case["op"] == "permute":                                              # x, dx; rows, their gradient; pos
        return {"bytes": 2.0 * h * (2 * t + 2 * t * kk) + 8 * t * kk, "flops": 1.0 * t * kk * h}
    return {"bytes": 2.0 * h * (2 * t + 2 * t * kk) + 16 * t * kk, "flops": 5.0 * t * kk * h}


# ------------------------------------------------------------------------------------------- inputs
def _group_sizes(rows, groups, active, seed):
    """Rows per expert as a router with logits ~ N(0, 0.5) gives them, over `active` experts with a row at least."""
    gen = torch.Generator().manual_seed(seed)
    who = torch.randperm(groups, generator=gen)[:active]
    sizes = torch.zeros(groups, dtype=torch.int64)
    sizes[who] = 1
    if rows > active:
        p = torch.softmax(0.5 * torch.randn(active, generator=gen), 0)
        more = torch.multinomial(p, rows - active, replacement=True, generator=gen)
        sizes[who] += torch.bincount(more, minlength=active)
    return sizes


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=DTYPES[case["dtype"]]):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype).mul_(std)

    if case["op"] == "gated_ffn":
        m, h, i, g = (case[k] for k in ("rows", "hidden", "inter", "groups"))
        sizes = _group_sizes(m, g, case["active"], seed)
        s = dict(case=case, sizes=sizes.cuda(), rows_per_group=sizes.tolist(), x=normal(m, h),
                 w13=normal(g, 2 * i, h, std=h ** -0.5), w2=normal(g, h, i, std=i ** -0.5))
        if case["train"]:
            s["dy"] = normal(m, h)
        return s
    if case["op"] == "w4":
        g, n, k, gs = (case[x] for x in ("groups", "n", "k", "group_size"))
        wn = 2 * n if case["gated"] else n
        sizes = _group_sizes(case["rows"], g, case["active"], seed)
        w4 = torch.randint(0, 256, (g, wn, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
        scale = normal(g, wn, k // gs, std=0.3).exp_().mul_(0.2 * k ** -0.5)
        zero = torch.randint(5, 11, (g, wn, k // gs), generator=gen, device="cuda", dtype=torch.uint8) if case["zero"] else None
        return dict(case=case, sizes=sizes.cuda(), rows_per_group=sizes.tolist(), a=normal(case["rows"], k), w4=w4, scale=scale,
                    zero=zero)
    t, kk, h = case["tokens"], case["top_k"], case["hidden"]
    expert = torch.topk(normal(t, 64, dtype=torch.float32), kk, dim=1).indices
    order = torch.argsort(expert.reshape(-1), stable=True)                   # pair in row r: rows sorted by expert
    pos = torch.empty_like(order)
    pos[order] = torch.arange(t * kk, device="cuda")                         # row of pair p
    s = dict(case=case, pos=pos, order=order)
    if case["op"] == "permute":
        return dict(s, x=normal(t, h), drows=normal(t * kk, h))
    weight = torch.softmax(normal(t, kk, dtype=torch.float32), 1)
    return dict(s, rows=normal(t * kk, h), weight=weight, dout=normal(t, h))


# ------------------------------------------------------------------------------------------- one pass
def run(state):
    return {"gated_ffn": _run_ffn, "w4": _run_w4, "permute": _run_permute, "combine": _run_combine}[state["case"]["op"]](state)


def _leaf(t):
    return t.detach().requires_grad_()


def _run_ffn(s):
    case = s["case"]
    if own:
        from triton_grouped_gemm_b200.gemm.autograd import grouped_gated_ffn

        if not case["train"]:
            return grouped_gated_ffn(s["x"], s["w13"], s["w2"], s["sizes"], activation=case["act"])
        x, w13, w2 = _leaf(s["x"]), _leaf(s["w13"]), _leaf(s["w2"])
        y = grouped_gated_ffn(x, w13, w2, s["sizes"], activation=case["act"])
        dx, dw13, dw2 = torch.autograd.grad(y, (x, w13, w2), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw13": dw13, "dw2": dw2}
    rows = s["rows_per_group"]
    xs = s["x"].split(rows)
    if not case["train"]:
        return torch.cat([_ffn_group(x, w13, w2, case["act"]) for x, w13, w2 in zip(xs, s["w13"], s["w2"]) if x.shape[0]])
    got = [_ffn_group_grad(x, w13, w2, dy, case["act"]) for x, w13, w2, dy in zip(xs, s["w13"], s["w2"], s["dy"].split(rows))]
    y, dx, dw13, dw2 = zip(*got)
    return {"y": torch.cat(y), "dx": torch.cat(dx), "dw13": torch.stack(dw13), "dw2": torch.stack(dw2)}


def _activation(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        p = torch.sigmoid(g)
        return g * p, p * (1 + g * (1 - p))
    c = math.sqrt(2 / math.pi)
    th = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + th), 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * c * (1 + 3 * 0.044715 * g * g)


def _ffn_group(x, w13, w2, act):
    g, u = (x.float() @ w13.float().T).chunk(2, dim=1)
    return ((_activation(g, act)[0] * u) @ w2.float().T).to(x.dtype)


def _ffn_group_grad(x, w13, w2, dy, act):
    dtype = x.dtype
    x, w13, w2, dy = x.float(), w13.float(), w2.float(), dy.float()
    g, u = (x @ w13.T).chunk(2, dim=1)
    a, slope = _activation(g, act)
    h, dh = a * u, dy @ w2
    dgu = torch.cat((dh * u * slope, dh * a), dim=1)
    return (h @ w2.T).to(dtype), (dgu @ w13).to(dtype), (dgu.T @ x).to(dtype), (dy.T @ h).to(dtype)


def _run_w4(s):
    case = s["case"]
    if own:
        from triton_grouped_gemm_b200.gemm.W4.m_grouped_gemm_w4 import m_grouped_gemm_w4, m_grouped_gemm_w4_gated

        b = (s["w4"], s["scale"], s["zero"])
        return m_grouped_gemm_w4_gated(s["a"], b, s["sizes"]) if case["gated"] else m_grouped_gemm_w4(s["a"], b, s["sizes"])
    zeros = s["zero"] if s["zero"] is not None else [None] * case["groups"]
    return torch.cat([_w4_group(a, w, sc, z, case["gated"])
                      for a, w, sc, z in zip(s["a"].split(s["rows_per_group"]), s["w4"], s["scale"], zeros) if a.shape[0]])


def _w4_group(a, w4, scale, zero, gated):
    q = torch.stack((w4 & 15, w4 >> 4), dim=-1).reshape(w4.shape[0], scale.shape[1], -1)   # [N, K / group, group]
    z = 8.0 if zero is None else zero.float().unsqueeze(-1)
    w = ((q.float() - z) * scale.float().unsqueeze(-1)).reshape(w4.shape[0], -1)
    c = a.float() @ w.T
    if gated:
        g, u = c.chunk(2, dim=1)
        c = g * torch.sigmoid(g) * u
    return c.to(a.dtype)


def _run_permute(s):
    kk = s["case"]["top_k"]
    if own:
        from triton_grouped_gemm_b200.ep.autograd import permute_rows

        x = _leaf(s["x"])
        rows = permute_rows(x, s["pos"], s["order"], kk)
        return {"rows": rows.detach(), "dx": torch.autograd.grad(rows, x, s["drows"])[0]}
    x, t = s["x"], s["x"].shape[0]
    dx = s["drows"][s["pos"]].view(t, kk, -1).float().sum(1).to(x.dtype)
    return {"rows": x[s["order"] // kk], "dx": dx}


def _run_combine(s):
    if own:
        from triton_grouped_gemm_b200.ep.autograd import combine_rows

        rows, weight = _leaf(s["rows"]), _leaf(s["weight"])
        out = combine_rows(rows, weight, s["pos"], s["order"])
        drows, dweight = torch.autograd.grad(out, (rows, weight), s["dout"])
        return {"out": out.detach(), "drows": drows, "dweight": dweight}
    t, kk = s["weight"].shape
    of_pair = s["rows"][s["pos"]].view(t, kk, -1).float()
    out = (of_pair * s["weight"].unsqueeze(-1)).sum(1).to(s["rows"].dtype)
    dout = s["dout"].float()
    dweight = (of_pair * dout.unsqueeze(1)).sum(-1)
    drows = (s["weight"].reshape(-1)[s["order"]].unsqueeze(-1) * dout[s["order"] // kk]).to(s["rows"].dtype)
    return {"out": out, "drows": drows, "dweight": dweight}


# ------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"gated_ffn": _exact_ffn, "w4": _exact_w4, "permute": _exact_permute, "combine": _exact_combine}[case["op"]](s)


def _exact_ffn(s):
    """The block written out in double precision; the gradients by differentiating that."""
    case, train = s["case"], s["case"]["train"]
    y = torch.empty(s["x"].shape, device="cuda", dtype=torch.float64)
    dx = torch.empty_like(y) if train else None
    dw13 = torch.zeros(s["w13"].shape, device="cuda", dtype=torch.float64) if train else None
    dw2 = torch.zeros(s["w2"].shape, device="cuda", dtype=torch.float64) if train else None
    lo = 0
    for e, rows in enumerate(s["rows_per_group"]):
        hi = lo + rows
        if rows:
            x, w13, w2 = (t.double().requires_grad_(train) for t in (s["x"][lo:hi], s["w13"][e], s["w2"][e]))
            gate, up = x.matmul(w13[:case["inter"]].t()), x.matmul(w13[case["inter"]:].t())
            if case["act"] == "silu":
                hid = gate / (1 + torch.exp(-gate)) * up
            else:
                hid = torch.nn.functional.gelu(gate, approximate="tanh") * up
            out = hid.matmul(w2.t())
            y[lo:hi] = out.detach()
            if train:
                dx[lo:hi], dw13[e], dw2[e] = torch.autograd.grad(out, (x, w13, w2), s["dy"][lo:hi].double())
        lo = hi
    return {"y": y, "dx": dx, "dw13": dw13, "dw2": dw2} if train else y


def _exact_w4(s):
    case, dev = s["case"], s["a"].device
    gs, k, n = case["group_size"], case["k"], case["n"]
    out = torch.empty(case["rows"], n, device=dev, dtype=torch.float64)
    column = torch.arange(k, device=dev)
    lo = 0
    for e, rows in enumerate(s["rows_per_group"]):
        if rows:
            byte = s["w4"][e][:, column // 2].to(torch.int64)
            q = torch.where(column % 2 == 0, byte % 16, byte // 16)
            z = s["zero"][e][:, column // gs].to(torch.int64) if s["zero"] is not None else 8
            w = (q - z).double() * s["scale"][e][:, column // gs].double()
            prod = torch.einsum("rk,nk->rn", s["a"][lo:lo + rows].double(), w)
            if case["gated"]:
                gate, up = prod[:, :n], prod[:, n:]
                prod = gate / (1 + torch.exp(-gate)) * up
            out[lo:lo + rows] = prod
        lo += rows
    return out


def _exact_permute(s):
    t, kk = s["case"]["tokens"], s["case"]["top_k"]
    dx = torch.zeros(t, s["case"]["hidden"], device="cuda", dtype=torch.float64)
    dx.index_add_(0, torch.div(s["order"], kk, rounding_mode="floor"), s["drows"].double())
    return {"rows": s["x"].double().repeat_interleave(kk, dim=0)[s["order"]], "dx": dx}


def _exact_combine(s):
    t, kk = s["weight"].shape
    token = torch.div(s["order"], kk, rounding_mode="floor")                 # of every row
    w = s["weight"].double().reshape(-1).gather(0, s["order"])
    rows, dout = s["rows"].double(), s["dout"].double().index_select(0, token)
    out = torch.zeros(t, s["case"]["hidden"], device="cuda", dtype=torch.float64)
    out.index_add_(0, token, rows * w.unsqueeze(1))
    dweight = torch.zeros(t * kk, device="cuda", dtype=torch.float64)
    dweight[s["order"]] = torch.linalg.vecdot(rows, dout)
    return {"out": out, "drows": dout * w.unsqueeze(1), "dweight": dweight.view(t, kk)}
