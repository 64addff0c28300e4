"""Workloads of the operators that train the experts, and of the dense 8-bit product.

Each case is one call of one operator. ``run`` computes it either in its plain form (elementary
torch operations in fp32, rounded once at the end) or, with ``own`` set, through the package's
entry points. ``exact`` computes the same from the definition in fp64.

Operators (``case["op"]``):
  grouped      y[r] = W[e] x[r], rows sorted by expert, any number for each
  grouped_bwd  its gradients: dx[r] = W[e]^T dy[r] and dW[e] = sum over e's rows of dy[r] x[r]^T
  silu         h = weight * silu(gate) * up, and an 8-bit copy of gate and up for the backward pass
  silu_bwd     its gradients from the 8-bit copy, with h computed again
  save         16-bit rows to 8 bits with a scale for each 128 columns, and back
  restore      such rows back to 16 bits in the order of an index (the experts' order of the tokens)
  int8         y = x W^T of int8 values with a scale for each row of x and of W

Sizes are those of the package's own configurations (H = 7168, I = 2048, E = 256, top-8; H = 4096,
I = 14336, E = 8, top-2; H = 1024, I = 512, E = 8; 64 experts with 9088 rows) and the ranges around them.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
Q_DTYPES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
GROUP = 128  # columns of one scale


def listed():
    return [
        # gate and up products of 64 tokens with 2 of 8 small experts: launch latency
        {"name": "grouped_r128", "op": "grouped", "R": 128, "E": 8, "N": 1024, "K": 1024, "dtype": "f16", "skew": 0.0, "rest": 0},
        # down products of 4096 tokens with 8 of 256 experts: 7.5 GB of weights, 128 rows for each on average
        {"name": "grouped_r32768", "op": "grouped", "R": 32768, "E": 256, "N": 7168, "K": 2048, "dtype": "bf16", "skew": 0.0,
         "rest": 0},
        # gradients of the down products of a ragged batch, unevenly routed to 8 large experts, some routes
        # dropped; the weights' gradient in fp32, as an optimiser's accumulator takes it
        {"name": "grouped_bwd_r4097", "op": "grouped_bwd", "R": 4097, "E": 8, "N": 4096, "K": 14336, "dtype": "bf16", "skew": 0.8,
         "rest": 33, "dw": "f32"},
        # gradients with 64 experts, some of them without rows
        {"name": "grouped_bwd_r9088", "op": "grouped_bwd", "R": 9088, "E": 64, "N": 7168, "K": 2048, "dtype": "f16", "skew": 1.2,
         "rest": 0, "dw": "f16"},
        # the activation of a small batch, with its copy for the backward pass
        {"name": "silu_r128", "op": "silu", "R": 128, "I": 512, "dtype": "bf16", "q": "int8", "weights": True},
        # the same for 4096 tokens with 8 experts each, e4m3
        {"name": "silu_r32768", "op": "silu", "R": 32768, "I": 2048, "dtype": "bf16", "q": "fp8", "weights": True},
        # the backward pass of the activation of as many rows, from int8
        {"name": "silu_bwd_r32768", "op": "silu_bwd", "R": 32768, "I": 2048, "dtype": "bf16", "q": "int8", "weights": True},
        # a ragged batch in fp16 without routing weights
        {"name": "silu_bwd_r2047", "op": "silu_bwd", "R": 2047, "I": 1000, "dtype": "f16", "q": "fp8", "weights": False},
        # a layer's input kept in 8 bits
        {"name": "save_t4096", "op": "save", "R": 4096, "H": 7168, "dtype": "bf16", "q": "int8"},
        # such an input restored for the weights' gradient: each token's row for each of its 8 experts
        {"name": "restore_r32768", "op": "restore", "T": 4096, "R": 32768, "H": 7168, "dtype": "bf16", "q": "int8"},
        # a dense projection (shared expert, H = 4096 to I = 14336) of one decoded token
        {"name": "int8_m1", "op": "int8", "M": 1, "N": 14336, "K": 4096, "out": "bf16", "bias": False},
        # the same of a prompt of odd length
        {"name": "int8_m4095", "op": "int8", "M": 4095, "N": 14336, "K": 4096, "out": "bf16", "bias": True},
    ]


def _log_int(rng, lo, hi):
    v = max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return v - 1 if v % 1024 == 0 and v > lo else v  # the listed cases have the round sizes


def _multiple(v, step):
    return max(step, v // step * step)


def draw(rng):
    op = rng.choice(["grouped", "grouped", "grouped_bwd", "grouped_bwd", "silu", "silu_bwd", "save", "restore", "int8", "int8",
                     "int8"])
    dtype = rng.choice(["f16", "bf16"])
    if op in ("grouped", "grouped_bwd"):
        E = rng.choice([1, 3, 8, 16, 60, 64, 128, 256])
        R = _log_int(rng, 1, 32768 if op == "grouped" else 9000)
        N, K = _multiple(_log_int(rng, 64, 14000), 8), _multiple(_log_int(rng, 64, 14000), 8)
        dw = rng.choice([dtype, "f32"])
        elements, products = (256 * 7168 * 2048, 32768 * 7168 * 2048) if op == "grouped" else (64 * 7168 * 2048, 9088 * 7168 * 2048)
        elements //= 2 if op == "grouped_bwd" and dw == "f32" else 1
        K = _multiple(min(K, elements // (E * N), products // (R * N)), 8)
        N = _multiple(min(N, elements // (E * K), products // (R * K)), 8)
        c = {"op": op, "R": R, "E": E, "N": N, "K": K, "dtype": dtype, "skew": rng.choice([0.0, 0.5, 1.2 if E < 128 else 0.3]),
             "rest": rng.choice([0, 0, rng.randint(0, min(R // 2, 40))])}
        if op == "grouped_bwd":
            c["dw"] = dw
        return c
    if op in ("silu", "silu_bwd"):
        I = _log_int(rng, 8, 14000)
        I = _multiple(I, 64) if rng.random() < 0.6 else I
        return {"op": op, "R": _log_int(rng, 1, min(32000, 32768 * 2048 // I)), "I": I, "dtype": dtype,
                "q": rng.choice(["int8", "fp8"]), "weights": rng.random() < 0.6}
    if op in ("save", "restore"):
        H = _log_int(rng, 8, 14000)
        H = _multiple(H, 64) if rng.random() < 0.6 else H
        T = _log_int(rng, 1, min(16000, 4096 * 7168 // H))
        c = {"op": op, "R": T, "H": H, "dtype": dtype, "q": rng.choice(["int8", "fp8"])}
        if op == "restore":
            c["T"], c["R"] = T, T * rng.randint(1, 8)
        return c
    N, K = _log_int(rng, 64, 16000), _multiple(_log_int(rng, 64, 14000), 16)
    out = rng.choice(["f16", "bf16", "f32"])
    most = min(8000, 4095 * 14336 * 4096 // (N * K), 4000 * 14336 * 2 // (N * (4 if out == "f32" else 2) + K))
    return {"op": op, "M": _log_int(rng, 1, most), "N": N, "K": K, "out": out, "bias": rng.random() < 0.4}


# ------------------------------------------------------------------------------------ inputs
def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _offsets(case, seed):
    """Numbers of rows of the experts as a router gives them: the expert of popularity rank i is chosen about
    i^-skew as often; the last ``rest`` rows belong to none."""
    E, rows = case["E"], case["R"] - case["rest"]
    rng = random.Random(seed)
    weights = [(i + 1) ** -case["skew"] * rng.uniform(0.7, 1.3) for i in range(E)]
    rng.shuffle(weights)
    sizes = [0] * E
    for e in rng.choices(range(E), weights, k=rows):
        sizes[e] += 1
    ends = [0]
    for n in sizes:
        ends.append(ends[-1] + n)
    return ends, max(sizes + [1])


def _q8(x, kind):
    """(values, scales) of rows x [R, W] fp32 whose values fit their 16-bit type: groups of 128 columns."""
    R, W = x.shape
    pad = -W % GROUP
    x = torch.nn.functional.pad(x, (0, pad)).view(R, -1, GROUP)
    amax = x.abs().amax(-1, keepdim=True)
    if kind == "int8":  # a division by a number would be a product with its rounded reciprocal
        most = torch.full_like(amax, 127)
        v = x * torch.where(amax > 0, most / amax, 0.0)
        q = (v.sign() * (v.abs() + 0.5).floor()).to(torch.int8)
        scale = amax / most
    else:  # the next power of two from amax / 448 on (448 = 0.875 * 2^9): no value is rounded but to e4m3
        m, e = torch.frexp(amax)
        scale = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), torch.where(m <= 0.875, e - 9, e - 8)), 0.0)
        q = (x / torch.where(amax > 0, scale, 1.0)).to(torch.float8_e4m3fn)
    return q.view(R, -1)[:, :W].contiguous(), scale.squeeze(-1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op == "int8":
        M, N, K = case["M"], case["N"], case["K"]
        for name, rows in (("x", M), ("w", N)):  # normal rows of different sizes, quantised row by row
            v = _randn(gen, rows, K)
            amax = v.abs().amax(-1, keepdim=True)
            s[name] = (v * (127 / amax)).round().to(torch.int8)
            size = 0.5 + torch.rand((rows,), generator=gen, device="cuda")
            s[name + "_scale"] = amax.squeeze(-1) / 127 * size * (1.0 if name == "x" else K ** -0.5)
        s["bias"] = _randn(gen, N) if case["bias"] else None
        return s
    dtype = DTYPES[case["dtype"]]
    if op in ("grouped", "grouped_bwd"):
        R, E, N, K = (case[n] for n in ("R", "E", "N", "K"))
        ends, s["most"] = _offsets(case, seed)
        s["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        s["x"] = _randn(gen, R, K).to(dtype)
        s["w"] = torch.empty((E, N, K), dtype=dtype, device="cuda").normal_(0, K ** -0.5, generator=gen)
        if op == "grouped_bwd":
            s["dy"] = _randn(gen, R, N).to(dtype)
        return s
    if op in ("silu", "silu_bwd"):
        R, I = case["R"], case["I"]
        gate_up = (1.5 * _randn(gen, R, 2 * I)).to(dtype)
        s["weights"] = torch.rand((R,), generator=gen, device="cuda") if case["weights"] else None
        if op == "silu":
            s["gate_up"] = gate_up
        else:  # gate and up have groups of their own
            q, scale = _q8(gate_up.float().view(2 * R, I), case["q"])
            s["q"], s["scale"] = q.view(R, 2 * I), scale.view(R, -1)
            s["dh"] = _randn(gen, R, I).to(dtype)
        return s
    T, H = case.get("T", case["R"]), case["H"]
    # the columns of a residual stream differ in size
    x = (_randn(gen, T, H) * torch.exp(0.5 * _randn(gen, H))).to(dtype)
    if op == "save":
        s["x"] = x
    else:
        s["q"], s["scale"] = _q8(x.float(), case["q"])
        s["index"] = torch.randperm(case["R"], generator=gen, device="cuda").remainder(T).to(torch.int32)
    return s


# ------------------------------------------------------------------------------------ the calls
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import muxi_race_b200 as m

    case = s["case"]
    op = case["op"]
    if op == "grouped":
        return m.grouped_linear(s["x"], s["w"], s["offsets"])
    if op == "grouped_bwd":
        dx, dw = m.grouped_linear_backward(s["dy"], s["x"], s["w"], s["offsets"], dw_dtype=DTYPES[case["dw"]])
        return {"dx": dx, "dw": dw}
    if op == "silu":
        h, saved = m.silu_mul_rows8(s["gate_up"], s["weights"], q_dtype=Q_DTYPES[case["q"]])
        return {"h": h, "gate_up": m.restore_rows8(saved), "scale": saved.scale}
    if op == "silu_bwd":
        saved = m.Rows8(s["q"], s["scale"], s["dh"].dtype, parts=2)
        dgate_up, dweights, h = m.silu_mul_backward(s["dh"], saved, s["weights"])
        return {"dgate_up": dgate_up, "dweights": dweights, "h": h}
    if op == "save":
        saved = m.save_rows8(s["x"], q_dtype=Q_DTYPES[case["q"]])
        return {"x": m.restore_rows8(saved), "scale": saved.scale}
    if op == "restore":
        return m.restore_rows8(m.Rows8(s["q"], s["scale"], DTYPES[case["dtype"]]), s["index"])
    return m.int8_linear(s["x"], s["x_scale"], s["w"], s["w_scale"], bias=s["bias"], out_dtype=DTYPES[case["out"]])


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op in ("grouped", "grouped_bwd"):
        return _plain_grouped(s)
    if op == "silu":
        R, I = case["R"], case["I"]
        x = s["gate_up"].float()
        g, u = x[:, :I], x[:, I:]
        h = g / (1 + torch.exp(-g)) * u
        h = h * s["weights"][:, None] if case["weights"] else h
        q, scale = _q8(x.view(2 * R, I), case["q"])
        back = _plain_restore(q, scale).view(R, 2 * I)
        return {"h": h.to(s["gate_up"].dtype), "gate_up": back.to(s["gate_up"].dtype), "scale": scale.view(R, -1)}
    if op == "silu_bwd":
        return _plain_silu_bwd(s)
    if op == "save":
        q, scale = _q8(s["x"].float(), case["q"])
        return {"x": _plain_restore(q, scale).to(s["x"].dtype), "scale": scale}
    if op == "restore":
        at = s["index"].long()
        return _plain_restore(s["q"][at], s["scale"][at]).to(DTYPES[case["dtype"]])
    # whole numbers below 2^24 in every product, above it in their sums: those are taken in parts that fit
    x, w = s["x"].float(), s["w"].float()
    parts = max(1, -(-case["K"] // 1024))
    pad = -case["K"] % parts
    x, w = (torch.nn.functional.pad(t, (0, pad)).view(t.shape[0], parts, -1).transpose(0, 1) for t in (x, w))
    y = torch.bmm(x, w.mT).to(torch.int32).sum(0).float() * s["x_scale"][:, None] * s["w_scale"]
    return (y if s["bias"] is None else y + s["bias"]).to(DTYPES[case["out"]])


def _plain_restore(q, scale):
    return q.float() * scale.repeat_interleave(GROUP, -1)[:, :q.shape[1]]


def _plain_grouped(s):
    """The experts' rows, each set padded to the largest, so that all products are one batched one."""
    case, ends, most = s["case"], s["offsets"].long(), s["most"]
    R, E = case["R"], case["E"]
    r = torch.arange(R, device="cuda")
    e = torch.searchsorted(ends, r, right=True) - 1  # E: a row of no expert
    inside = (e < E)[:, None]
    slot = torch.where(inside[:, 0], e * most + r - ends[e.clamp_max(E - 1)], E * most)

    def spread(t):
        p = torch.zeros((E * most + 1, t.shape[1]), dtype=torch.float32, device="cuda")
        p[slot] = t.float()
        return p[:-1].view(E, most, -1)

    def rows(p):
        return (p.reshape(E * most, -1)[slot.clamp_max(E * most - 1)] * inside).to(s["x"].dtype)

    w, x = s["w"].float(), s["x"]
    if case["op"] == "grouped":
        return rows(torch.bmm(spread(x), w.mT))
    x = spread(torch.where(inside, x, 0))
    dy = spread(torch.where(inside, s["dy"], 0))
    return {"dx": rows(torch.bmm(dy, w)), "dw": torch.bmm(dy.mT, x).to(DTYPES[case["dw"]])}


def _plain_silu_bwd(s):
    case, dh = s["case"], s["dh"].float()
    R, I = case["R"], case["I"]
    x = _plain_restore(s["q"].view(2 * R, I), s["scale"].view(2 * R, -1)).view(R, 2 * I)
    g, u = x[:, :I], x[:, I:]
    sig = 1 / (1 + torch.exp(-g))
    act = g * sig
    weights = s["weights"][:, None] if case["weights"] else 1.0
    dg = dh * weights * u * (sig * (1 + g * (1 - sig)))
    du = dh * weights * act
    return {"dgate_up": torch.cat((dg, du), -1).to(s["dh"].dtype),
            "dweights": (dh * act * u).sum(-1) if case["weights"] else None, "h": (weights * act * u).to(s["dh"].dtype)}


# ------------------------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    if op in ("grouped", "grouped_bwd"):
        R, E, N, K = (case[n] for n in ("R", "E", "N", "K"))
        rows = R - case["rest"]
        total = sum((i + 1) ** -case["skew"] for i in range(E))
        active = sum(1 - (1 - (i + 1) ** -case["skew"] / total) ** rows for i in range(E))  # experts with rows, as expected
        if op == "grouped":
            return {"bytes": 2 * (active * N * K + rows * K + R * N), "flops": 2 * rows * N * K}
        return {"bytes": 2 * (active * N * K + rows * (N + K) + R * K) + E * N * K * (4 if case["dw"] == "f32" else 2),
                "flops": 4 * rows * N * K}
    if op in ("silu", "silu_bwd"):
        R, I = case["R"], case["I"]
        copy = 2 * R * I + 8 * R * -(-I // GROUP)
        # forward: gate_up, h, the copy, and the copy read back into 16 bits; backward: the copy, dh, dgate_up, h
        return {"bytes": (4 + 2 + 4) * R * I + 2 * copy + 4 * R if op == "silu" else (2 + 4 + 2) * R * I + copy + 8 * R,
                "flops": (8 if op == "silu" else 20) * R * I}
    if op in ("save", "restore"):
        R, H = case["R"], case["H"]
        T = case.get("T", R)
        copy = T * H + 4 * T * -(-H // GROUP)
        return {"bytes": 4 * R * H + 2 * copy if op == "save" else 2 * R * H + 4 * R + copy, "flops": 3 * R * H}
    M, N, K = case["M"], case["N"], case["K"]
    return {"bytes": M * K + N * K + M * N * (4 if case["out"] == "f32" else 2) + 4 * (M + N * (2 if case["bias"] else 1)),
            "flops": 2 * M * N * K}


# ------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    f = lambda t: t.to(torch.float64)  # noqa: E731

    def encode(x):
        """The values that 8 bits stand for, and the scales, of fp64 rows whose values fit 16 bits."""
        v = torch.zeros(x.shape[0], -(-x.shape[1] // GROUP) * GROUP, dtype=torch.float64, device="cuda")
        v[:, :x.shape[1]] = x
        v = v.unflatten(1, (-1, GROUP))
        top = v.abs().amax(2)
        if case["q"] == "int8":
            scale = top / torch.full_like(top, 127)
            code = v / scale.clamp_min(1e-300)[..., None]
            code = torch.sign(code) * torch.floor(code.abs() + 0.5)
        else:
            scale = torch.ldexp(torch.ones_like(top), torch.log2(top.clamp_min(1e-300) / 448).floor().int() - 1)
            for _ in range(3):  # the first power of two that is large enough
                scale = torch.where(448 * scale < top, 2 * scale, scale)
            scale = torch.where(top > 0, scale, 0.0)
            code = v / scale.clamp_min(1e-300)[..., None]
            step = 2 ** (torch.floor(torch.log2(code.abs().clamp_min(2.0 ** -6))) - 3)
            code = torch.round(code / step) * step
        return (code * scale[..., None]).flatten(1)[:, :x.shape[1]], scale

    def decode(q, scale):
        columns = torch.arange(q.shape[1], device="cuda") // GROUP
        return f(q.float()) * f(scale)[:, columns]

    if op in ("grouped", "grouped_bwd"):
        ends = s["offsets"].tolist()
        spans = [(e, slice(ends[e], ends[e + 1])) for e in range(case["E"]) if ends[e] < ends[e + 1]]
        if op == "grouped":
            y = torch.zeros(case["R"], case["N"], dtype=torch.float64, device="cuda")
            for e, at in spans:
                y[at] = f(s["x"][at]) @ f(s["w"][e]).T
            return y
        dx = torch.zeros(case["R"], case["K"], dtype=torch.float64, device="cuda")
        dw = torch.zeros(case["E"], case["N"], case["K"], dtype=torch.float64, device="cuda")
        for e, at in spans:
            dy = f(s["dy"][at])
            dx[at] = dy @ f(s["w"][e])
            dw[e] = dy.T @ f(s["x"][at])
        return {"dx": dx, "dw": dw}
    if op == "silu":
        g, u = f(s["gate_up"]).chunk(2, 1)
        h = torch.sigmoid(g) * g * u
        if s["weights"] is not None:
            h = h * f(s["weights"]).unsqueeze(1)
        (qg, sg), (qu, su) = encode(g), encode(u)
        return {"h": h, "gate_up": torch.cat((qg, qu), 1), "scale": torch.cat((sg, su), 1)}
    if op == "silu_bwd":
        I, groups = case["I"], s["scale"].shape[1] // 2
        g = decode(s["q"][:, :I], s["scale"][:, :groups]).requires_grad_()
        u = decode(s["q"][:, I:], s["scale"][:, groups:]).requires_grad_()
        w = (torch.ones(case["R"], device="cuda") if s["weights"] is None else s["weights"]).to(torch.float64).requires_grad_()
        h = torch.nn.functional.silu(g) * u * w[:, None]
        dg, du, dw = torch.autograd.grad((h * f(s["dh"])).sum(), (g, u, w))
        return {"dgate_up": torch.cat((dg, du), 1), "dweights": None if s["weights"] is None else dw, "h": h.detach()}
    if op == "save":
        x, scale = encode(f(s["x"]))
        return {"x": x, "scale": scale}
    if op == "restore":
        return decode(s["q"], s["scale"])[s["index"].long()]
    y = (f(s["x"]) @ f(s["w"]).T) * f(s["x_scale"])[:, None] * f(s["w_scale"])[None]
    return y if s["bias"] is None else y + f(s["bias"])
