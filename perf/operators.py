"""Cases, plain forms and exact values of the operators around the head: the residual addition with
its RMSNorm (training, and with an e4m3 output for 8-bit products), the gated projection of a
feed-forward block (training, single tokens, and on e4m3 operands), and the clipping of gradients by
their global norm.

``run`` computes the plain form in 32-bit torch operations, or calls ``rus_b200`` where ``own`` is
set; ``exact`` computes the definition in 64 bits. Sizes are those of the heads the benchmark knows
(hidden 896, 1536, 3584, 4096 with their models' feed-forward widths and packed token counts).
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------- cases ---


def listed():
    return [
        # one new token of a 0.5B model between two sub-layers: latency only
        dict(name="norm token", op="norm", rows=1, hidden=896, dtype="float16", train=False),
        # 4 packed rows of 512 tokens, fine-tuning a 1.5B model
        dict(name="norm train 2048x1536", op="norm", rows=2048, hidden=1536, dtype="float16", train=True),
        # 8 x 4096 tokens of an 8B model, the longest training batch
        dict(name="norm train 32768x4096", op="norm", rows=32768, hidden=4096, dtype="bfloat16", train=True),
        # a decoding batch of a 7B model whose projections run in 8 bits
        dict(name="norm e4m3 64x3584", op="norm_e4m3", rows=64, hidden=3584, dtype="bfloat16"),
        # the prefill of a packed batch of the same model
        dict(name="norm e4m3 9434x3584", op="norm_e4m3", rows=9434, hidden=3584, dtype="bfloat16"),
        # one new token of a 1.5B model: the weights' read is all there is
        dict(name="gated token 1536x8960", op="gated", rows=1, hidden=1536, ffn=8960, dtype="bfloat16", act="silu",
             train=False),
        # the reference's real call: a packed batch of 693 tokens, forward and backward
        dict(name="gated train 693x1536x8960", op="gated", rows=693, hidden=1536, ffn=8960, dtype="float16",
             act="silu", train=True),
        # two rows of 4096 tokens of an 8B model, forward and backward
        dict(name="gated train 8192x4096x14336", op="gated", rows=8192, hidden=4096, ffn=14336, dtype="bfloat16",
             act="silu", train=True),
        # a decoding batch of a 7B model on e4m3 weights
        dict(name="gated e4m3 64x3584x18944", op="gated_e4m3", rows=64, hidden=3584, ffn=18944, dtype="bfloat16",
             act="silu"),
        # the prefill of a packed batch on e4m3 weights
        dict(name="gated e4m3 9434x3584x18944", op="gated_e4m3", rows=9434, hidden=3584, ffn=18944,
             dtype="bfloat16", act="silu"),
        # low-rank adapters of a 1.5B model, 392 small fp32 gradients packed back to back as in communication buckets
        dict(name="clip adapters", op="clip", kind="adapter", layers=28, hidden=1536, ffn=8960, kv=256, rank=16,
             vocab=0, dtype="float32", align=1, clipped=True),
        # every gradient of a 0.5B model, 16-bit weights and fp32 norms
        dict(name="clip full 0.5B", op="clip", kind="full", layers=24, hidden=896, ffn=4864, kv=128, rank=0,
             vocab=151936, dtype="bfloat16", align=256, clipped=True),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    op = rng.choice(["norm", "norm_e4m3", "gated", "gated", "gated_e4m3", "clip"])
    dtype = rng.choice(["float16", "bfloat16"])
    act = rng.choice(["silu", "silu", "gelu_tanh"])
    if op in ("norm", "norm_e4m3"):
        hidden = 8 * round(_log(rng, 256, 8192) / 8)
        rows = int(_log(rng, 1, min(32768, 32768 * 4096 // hidden)))
        case = dict(op=op, rows=rows, hidden=hidden, dtype=dtype)
        return dict(case, train=rng.random() < 0.7) if op == "norm" else case
    if op in ("gated", "gated_e4m3"):
        step = 64 if op == "gated" else 128
        hidden = step * max(2, round(_log(rng, 256, 5120) / step))
        ffn = 64 * round(_log(rng, 512, 18944) / 64)
        rows = int(_log(rng, 1, min(16384, 8192 * 4096 * 14336 // (hidden * ffn))))
        case = dict(op=op, rows=rows, hidden=hidden, ffn=ffn, dtype=dtype, act=act)
        return dict(case, train=rng.random() < 0.7) if op == "gated" else case
    kind = rng.choice(["adapter", "full"])
    hidden = 64 * round(_log(rng, 256, 1536) / 64)
    return dict(op="clip", kind=kind, layers=rng.randint(1, 28 if kind == "adapter" else 12), hidden=hidden,
                ffn=64 * round(hidden * rng.uniform(2, 6) / 64), kv=64 * rng.randint(1, 4),
                rank=rng.randint(1, 64) if kind == "adapter" else 0,
                vocab=0 if kind == "adapter" else rng.randint(1000, 120000), dtype=rng.choice(sorted(DTYPES)),
                align=rng.choice([1, 256]), clipped=rng.random() < 0.7)


def _clip_shapes(c):
    """(shape, is a norm weight) of every gradient, in the order of the model's parameters."""
    h, f, kv, r = c["hidden"], c["ffn"], c["kv"], c["rank"]
    linears = [(h, h), (kv, h), (kv, h), (h, h), (f, h), (f, h), (h, f)]
    shapes = [((c["vocab"], h), False)] if c["vocab"] else []
    for _ in range(c["layers"]):
        if c["kind"] == "adapter":
            shapes += [s for o, i in linears for s in (((r, i), False), ((o, r), False))]
        else:
            shapes += [((o, i), False) for o, i in linears] + [((h,), True), ((h,), True)]
            shapes += [((h,), False), ((kv,), False), ((kv,), False)]  # the q, k and v biases
    return shapes


def work(case):
    op = case["op"]
    if op == "clip":
        size = {"float32": 4}.get(case["dtype"], 2)
        total = sum(math.prod(s) * (4 if norm else size) for s, norm in _clip_shapes(case))
        values = sum(math.prod(s) for s, _ in _clip_shapes(case))
        # read once, and written once where they are clipped
        return {"bytes": total * (2 if case["clipped"] else 1), "flops": (3 if case["clipped"] else 2) * values}
    n, h = case["rows"], case["hidden"]
    if op == "norm":
        # x, residual -> y, s; with training dy, ds -> dx (which is both inputs' gradient), dweight
        return {"bytes": 2 * n * h * (7 if case["train"] else 4) + 2 * h * (2 if case["train"] else 1),
                "flops": n * h * (13 if case["train"] else 5)}
    if op == "norm_e4m3":
        return {"bytes": n * h * 7 + 2 * h + 4 * n, "flops": 7 * n * h}
    f = case["ffn"]
    if op == "gated_e4m3":
        return {"bytes": n * h + 2 * f * h + 2 * n * f + 4 * n + 8 * f, "flops": 4 * n * h * f}
    if not case["train"]:
        return {"bytes": 2 * (n * h + 2 * f * h + n * f), "flops": 4 * n * h * f}
    # x, both weights, dh in; h, dx and both weight gradients out
    return {"bytes": 2 * (2 * n * h + 4 * f * h + 2 * n * f), "flops": 12 * n * h * f}


# ------------------------------------------------------------------ inputs ---


def _randn(gen, *shape, scale=1.0):
    return torch.randn(*shape, device="cuda", generator=gen).mul_(scale)


def _rows_e4m3(w):
    """Rows of w in e4m3 with one scale each, as a program keeps its weights for 8-bit products."""
    scale = w.abs().amax(dim=-1) / E4M3_MAX
    return (w / scale[:, None]).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    dt = DTYPES[case["dtype"]]
    op = case["op"]
    if op == "clip":
        shapes = _clip_shapes(case)
        grads, params, flats, fresh = [], [], [], []
        for norms in (False, True):
            some = [s for s, norm in shapes if norm == norms]
            if not some:
                continue
            t = torch.float32 if norms else dt
            align = case["align"]
            starts, total = [], 0
            for s in some:
                starts.append(total)
                total += -(-math.prod(s) // align) * align
            flat = torch.empty(total, device="cuda", dtype=t)
            flat.normal_(generator=gen).mul_(2e-3)
            for s, a in zip(some, starts):  # nothing between two gradients
                flat[a + math.prod(s):a + -(-math.prod(s) // align) * align].zero_()
            flats.append(flat)
            fresh.append(flat.clone())
            weights = torch.zeros(total, device="cuda", dtype=t)
            for s, a in zip(some, starts):
                p = weights[a:a + math.prod(s)].view(s).requires_grad_(True)
                p.grad = flat[a:a + math.prod(s)].view(s)
                params.append(p)
                grads.append(p.grad)
        count = sum(math.prod(s) for s, _ in shapes)
        norm = 2e-3 * math.sqrt(count)
        return dict(state, params=params, grads=grads, flats=flats, fresh=fresh,
                    max_norm=norm * (0.3 if case["clipped"] else 3.0))
    n, h = case["rows"], case["hidden"]
    # a residual stream: channels of very different size, a few of them large
    channel = torch.exp(_randn(gen, h, scale=0.5))
    channel[torch.randint(0, h, (max(1, h // 500),), device="cuda", generator=gen)] *= 20.0
    if op in ("norm", "norm_e4m3"):
        state["x"] = _randn(gen, n, h, scale=0.3).to(dt)
        state["residual"] = (_randn(gen, n, h) * channel).to(dt)
        state["weight"] = (1 + _randn(gen, h, scale=0.1)).to(dt)
        if case.get("train"):
            state["dy"] = _randn(gen, n, h, scale=1e-2).to(dt)
            state["ds"] = _randn(gen, n, h, scale=1e-2).to(dt)
            for name in ("x", "residual", "weight"):
                state[name].requires_grad_(True)
        return state
    f = case["ffn"]
    x = _randn(gen, n, h)
    gate, up = _randn(gen, f, h, scale=1.5 / math.sqrt(h)), _randn(gen, f, h, scale=1.0 / math.sqrt(h))
    if op == "gated_e4m3":
        state["x"], state["x_scale"] = _rows_e4m3(x)
        state["gate"], state["gate_scale"] = _rows_e4m3(gate)
        state["up"], state["up_scale"] = _rows_e4m3(up)
        return state
    state.update(x=x.to(dt), gate=gate.to(dt), up=up.to(dt))
    if case["train"]:
        state["dh"] = _randn(gen, n, f, scale=1e-2).to(dt)
        for name in ("x", "gate", "up"):
            state[name].requires_grad_(True)
    return state


# --------------------------------------------------------------------- run ---


def _act(g, kind):
    """(activation, its derivative)."""
    if kind == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)


def _plain_norm(st, train):
    x, r, w = st["x"].detach(), st["residual"].detach(), st["weight"].detach()
    s = (x.float() + r.float()).to(x.dtype)  # the residual stream is held, and normed, in the inputs' type
    v, wf = s.float(), w.float()
    rstd = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    norm = v * rstd
    y = norm * wf
    if not train:
        return y, s
    dy, ds = st["dy"].float(), st["ds"].float()
    p = dy * wf
    dx = ((p - norm * (p * norm).mean(-1, keepdim=True)) * rstd + ds).to(x.dtype)
    return y.to(x.dtype), s, dx, dx, (dy * norm).sum(0).to(w.dtype)


def _plain_gated(st, case):
    x, gate, up = (st[k].detach() for k in ("x", "gate", "up"))
    xf, gf, uf = x.float(), gate.float(), up.float()
    g, u = xf @ gf.T, xf @ uf.T
    if case["op"] == "gated_e4m3":
        g = g * st["x_scale"][:, None] * st["gate_scale"]
        u = u * st["x_scale"][:, None] * st["up_scale"]
    a, da = _act(g, case["act"])
    h = (a * u).to(DTYPES[case["dtype"]])
    if not case.get("train"):
        return h
    dh = st["dh"].float()
    dg, du = dh * u * da, dh * a
    return (h, (dg @ gf + du @ uf).to(x.dtype), (dg.T @ xf).to(gate.dtype), (du.T @ xf).to(up.dtype))


def _plain_clip(st):
    total = torch.stack([g.float().square().sum(dtype=torch.float64) for g in st["grads"]]).sum().sqrt().float()
    coef = (st["max_norm"] / (total + 1e-6)).clamp(max=1.0)
    for g in st["grads"]:
        g.copy_(g.float() * coef)
    return total


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        import rus_b200
    if op == "clip":
        if case["clipped"]:
            for flat, fresh in zip(state["flats"], state["fresh"]):
                flat.copy_(fresh)  # stands for the backward pass that writes the gradients of each step
        total = rus_b200.clip_grad_norm_(state["params"], state["max_norm"]) if own else _plain_clip(state)
        return [total] + state["flats"]
    if op == "norm":
        if not own:
            out = _plain_norm(state, case["train"])
            return out if case["train"] else (out[0].to(out[1].dtype), out[1])
        x, r, w = state["x"], state["residual"], state["weight"]
        y, s = rus_b200.add_rms_norm(x, r, w, EPS)
        if not case["train"]:
            return y, s
        return (y.detach(), s.detach(), *torch.autograd.grad((y, s), (x, r, w), (state["dy"], state["ds"])))
    if op == "norm_e4m3":
        if own:
            return rus_b200.add_rms_norm_e4m3(state["x"], state["residual"], state["weight"], EPS)
        y, s = _plain_norm(state, False)
        scale = y.abs().amax(-1) / E4M3_MAX
        scale = torch.where(scale > 0, scale, 1.0)
        return (y / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale, s
    if not own:
        return _plain_gated(state, case)
    if op == "gated_e4m3":
        return rus_b200.gated_linear_e4m3(state["x"], state["x_scale"], state["gate"], state["gate_scale"],
                                          state["up"], state["up_scale"], case["act"], DTYPES[case["dtype"]])
    x, gate, up = state["x"], state["gate"], state["up"]
    h = rus_b200.gated_linear(x, gate, up, case["act"])
    if not case["train"]:
        return h
    return (h.detach(), *torch.autograd.grad(h, (x, gate, up), state["dh"]))


# ------------------------------------------------------------------- exact ---


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "clip":
        total = math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in st["grads"]))
        k = min(1.0, st["max_norm"] / (total + 1e-6))
        return [torch.tensor(total, dtype=torch.float64)] + [t.double() * k for t in st["fresh"]]
    x = st["x"].detach().double()
    if op in ("norm", "norm_e4m3"):
        s = x + st["residual"].detach().double()
        held = s.to(st["x"].dtype).double()
        w = st["weight"].detach().double()
        inv = 1.0 / torch.sqrt((held * held).sum(-1, keepdim=True) / held.shape[-1] + EPS)
        y = held * inv * w
        if op == "norm_e4m3":
            top = y.abs().max(-1).values / E4M3_MAX
            top[top == 0] = 1.0
            return y / top[:, None], top, s
        if not case["train"]:
            return y, s
        dy = st["dy"].double()
        q = dy * w
        mean = (q * held).sum(-1, keepdim=True) / held.shape[-1]
        dx = st["ds"].double() + inv * q - held * inv ** 3 * mean
        return y, s, dx, dx, (dy * held * inv).sum(0)
    if op == "gated_e4m3":
        x = x * st["x_scale"].double()[:, None]
        wg = st["gate"].double() * st["gate_scale"].double()[:, None]
        wu = st["up"].double() * st["up_scale"].double()[:, None]
    else:
        wg, wu = st["gate"].detach().double(), st["up"].detach().double()
    g, u = torch.mm(x, wg.t()), torch.mm(x, wu.t())
    if case["act"] == "silu":
        sig = torch.sigmoid(g)
        a, da = g * sig, sig + g * sig * (1.0 - sig)
    else:
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * g + c * 0.044715 * g ** 3)
        a = g * (0.5 + 0.5 * t)
        da = 0.5 + 0.5 * t + g * 0.5 * (1.0 - t ** 2) * (c + 3.0 * c * 0.044715 * g ** 2)
    if not case.get("train"):
        return a * u
    dh = st["dh"].double()
    du = dh * a
    dg = dh * u * da
    return a * u, torch.mm(dg, wg) + torch.mm(du, wu), torch.mm(dg.t(), x), torch.mm(du.t(), x)
