"""Workloads of the operators around the expert MLP: normalisation, routing and 4-bit products.

Each case is one call of one operator. ``run`` computes it either in its plain form (elementary
torch operations in fp32, rounded once at the end) or, with ``own`` set, through the package's
entry points. ``exact`` computes the same from the definition in fp64.

Operators (``case["op"]``):
  norm        y = rms_norm(x + residual) * weight and the sum, optionally with 8-bit output rows
  norm_bwd    gradients of the norm for x (= residual) and weight
  route       top-k routing of router logits to expert ids, weights and per-expert counts
  route_bwd   gradient of the routing weights for the logits
  linear      y = x W^T with 4-bit weights in groups along K
  experts     the routed expert MLP with 4-bit weights

Sizes are those of the package's own configurations (H = 7168, I = 2048, E = 256, top-8; H = 4096,
I = 14336, E = 8, top-2; 1 to 32768 tokens) and the ranges around them.
"""
import math

import torch

own = False

EPS = 1e-6
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
Q_DTYPES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
Q_MAX = {"int8": 127.0, "fp8": 448.0}
NEG_INF = float("-inf")


def listed():
    return [
        # one decode step of one sequence: the norm between attention and experts; launch latency
        {"name": "norm_t1", "op": "norm", "T": 1, "H": 7168, "dtype": "bf16", "weight": "bf16", "residual": True,
         "quant": "none"},
        # a prompt's norm that feeds 8-bit experts: one pass over x and residual
        {"name": "norm_fp8_t4096", "op": "norm", "T": 4096, "H": 7168, "dtype": "bf16", "weight": "bf16",
         "residual": True, "quant": "fp8"},
        # a decode batch of odd size that feeds int8 experts, fp32 norm weights, no residual stream
        {"name": "norm_int8_t129", "op": "norm", "T": 129, "H": 4096, "dtype": "f16", "weight": "f32",
         "residual": False, "quant": "int8"},
        # a training micro-batch with a ragged number of tokens: gradient of the norm with the
        # residual branch's gradient added
        {"name": "norm_bwd_t8191", "op": "norm_bwd", "T": 8191, "H": 4096, "dtype": "bf16", "weight": "f32",
         "residual": True},
        # a decode batch through a sigmoid router with balance bias and groups (256 experts, 8 groups)
        {"name": "route_t128", "op": "route", "T": 128, "E": 256, "k": 8, "dtype": "f32", "scoring": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "renorm": True, "scale": 2.5, "masked": 0.0},
        # the largest prompt batch of the expert-parallel configuration, softmax scores kept as they
        # are, some experts switched off for some tokens
        {"name": "route_t32768", "op": "route", "T": 32768, "E": 256, "k": 8, "dtype": "f32", "scoring": "softmax",
         "bias": False, "groups": 1, "top_groups": 1, "renorm": False, "scale": 1.0, "masked": 0.05},
        # the same batch in training: dense gradient rows
        {"name": "route_bwd_t32768", "op": "route_bwd", "T": 32768, "E": 256, "k": 8, "dtype": "f32",
         "scoring": "softmax", "bias": False, "groups": 1, "top_groups": 1, "renorm": False, "scale": 1.0,
         "masked": 0.0},
        # a dense projection (shared expert, H = 4096 to I = 14336) for a single token
        {"name": "linear_t1", "op": "linear", "M": 1, "N": 14336, "K": 4096, "group": 128, "zeros": False,
         "dtype": "f16"},
        # an output projection for a small decode batch, fine groups with zero points
        {"name": "linear_t17", "op": "linear", "M": 17, "N": 7168, "K": 14336, "group": 32, "zeros": True,
         "dtype": "bf16"},
        # one token through its 8 of 256 experts
        {"name": "experts_t1", "op": "experts", "T": 1, "H": 7168, "I": 2048, "E": 64, "k": 8, "group": 128,
         "zeros": False, "dtype": "f16", "skew": 0.0},
        # a decode batch of 128 tokens over all 256 experts: the expert weights stream once
        {"name": "experts_t128", "op": "experts", "T": 128, "H": 7168, "I": 2048, "E": 256, "k": 8, "group": 128,
         "zeros": False, "dtype": "f16", "skew": 0.0},
        # few large experts, unevenly loaded, an odd batch: many tokens per expert
        {"name": "experts_e8_t33", "op": "experts", "T": 33, "H": 4096, "I": 14336, "E": 8, "k": 2, "group": 64,
         "zeros": True, "dtype": "bf16", "skew": 1.1},
    ]


def _log_int(rng, lo, hi):
    v = max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return v - 1 if v % 1024 == 0 and v > lo else v  # the listed cases have the round sizes


def _log_multiple(rng, lo, hi, step):
    """Mostly an odd multiple of `step`, as sizes of models are multiples; otherwise any size."""
    v = _log_int(rng, lo, hi)
    return max(lo, (v // step | 1) * step) if rng.random() < 0.7 and v >= 2 * step else v


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_bwd", "route", "route_bwd", "linear", "linear", "experts", "experts"])
    if op in ("norm", "norm_bwd"):
        dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
        H = _log_multiple(rng, 64, 16000, 64)
        c = {"op": op, "T": _log_int(rng, 1, 8192), "H": H, "dtype": dtype,
             "weight": rng.choice([dtype, "f32"]), "residual": rng.random() < 0.7}
        if op == "norm":
            c["quant"] = rng.choice(["none", "none", "int8", "fp8"]) if dtype != "f32" else "none"
        return c
    if op in ("route", "route_bwd"):
        groups = rng.choice([1, 1, 4, 8])
        E = groups * max(2, _log_int(rng, 8, 512) // groups)
        top_groups = 1 if groups == 1 else rng.randint(groups // 2, groups)
        k = rng.randint(1, min(8, top_groups * (E // groups)))
        return {"op": op, "T": _log_int(rng, 1, 32768), "E": E, "k": k,
                "dtype": rng.choice(["f32", "f32", "f16", "bf16"]), "scoring": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups,
                # a single renormalised weight is a constant
                "renorm": k > 1 and rng.random() < 0.6, "scale": rng.choice([1.0, 2.5]),
                "masked": rng.choice([0.0, 0.0, 0.3])}
    group = rng.choice([32, 64, 128, 128])
    zeros = rng.random() < 0.5
    dtype = rng.choice(["f16", "bf16"])
    if op == "linear":
        K, N = _log_multiple(rng, 64, 16000, 128), _log_multiple(rng, 64, 16000, 16)
        return {"op": op, "M": _log_int(rng, 1, 48), "N": N, "K": K, "group": group, "zeros": zeros, "dtype": dtype}
    E = rng.choice([8, 16, 32, 60, 64])
    H = (_log_int(rng, 256, 7000) // 64 | 1) * 64
    I = _log_multiple(rng, 128, min(4000, 7168 * 2048 // H - 64), 64)
    return {"op": op, "T": _log_int(rng, 1, 128), "H": H, "I": I, "E": E, "k": rng.choice([1, 2, 4, 8]),
            "group": group, "zeros": zeros, "dtype": dtype, "skew": rng.choice([0.0, 0.0, 1.1])}


# ------------------------------------------------------------------------------------ inputs
def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _route_scores64(logits, scoring):
    """fp64 scores, 0 where the logit is -inf."""
    l = logits.double()
    if scoring == "sigmoid":
        return torch.sigmoid(l)
    m = l.amax(-1, keepdim=True)
    e = torch.exp(l - torch.where(m == NEG_INF, 0.0, m))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-300)


def _near_ties(case, logits, bias):
    """Rows of `logits` where two candidates of the selection are nearer than fp32 can tell apart."""
    T, E, k, n = case["T"], case["E"], case["k"], case["groups"]
    c = _route_scores64(logits, case["scoring"])
    if bias is not None:
        c = c + bias.double()
    c = c.masked_fill(logits.double() == NEG_INF, NEG_INF)

    def close(v, count):
        v = v.sort(dim=-1, descending=True).values[:, :count + 1]
        gap = v[:, :-1] - v[:, 1:]
        return ((gap > 0) & (gap < 4e-6 * v[:, :-1].abs().clamp_min(1e-3))).any(-1)

    bad = torch.zeros(T, dtype=torch.bool, device=logits.device)
    if n > 1:
        score = c.view(T, n, E // n).sort(dim=-1, descending=True).values[..., :2].sum(-1)
        bad |= close(score, case["top_groups"])
        best = score.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros(T, n, dtype=torch.bool, device=logits.device).scatter_(1, best, True)
        c = c.masked_fill(~keep.repeat_interleave(E // n, 1), NEG_INF)
    return bad | close(c, k)


def _route_inputs(case, gen):
    T, E = case["T"], case["E"]
    # the balance bias is moved by steps of 0.001 in training
    bias = torch.randint(-40, 41, (E,), generator=gen, device="cuda").float() * 1e-3 if case["bias"] else None

    def logits_of(rows):
        l = _randn(gen, rows, E) * 1.5
        if case["masked"]:
            l = l.masked_fill(torch.rand((rows, E), generator=gen, device="cuda") < case["masked"], NEG_INF)
        return l.to(DTYPES[case["dtype"]])

    logits = logits_of(T)
    # Two forms of an fp32 score differ in the last bits, so a choice between scores that near has
    # no right answer: the few such rows are drawn again.
    for _ in range(20):
        bad = _near_ties(case, logits, bias)
        if not bool(bad.any()):
            break
        logits[bad] = logits_of(int(bad.sum()))
    if case["masked"] and T > 2:
        logits[T // 2] = NEG_INF  # a token without any expert
    return logits, bias


def _w4_inputs(gen, lead, N, K, group, zeros, dtype):
    """4-bit values two to a byte (low half first), scales and zero points of weights ~ N(0, 1/K)."""
    G = -(-K // group)
    q = torch.randint(0, 256, (*lead, N, (K + 1) // 2), generator=gen, device="cuda", dtype=torch.uint8)
    s = (torch.rand((*lead, N, G), generator=gen, device="cuda") + 0.5) * (0.2 * K ** -0.5)
    z = torch.randint(4, 12, (*lead, N, G), generator=gen, device="cuda", dtype=torch.uint8) if zeros else None
    return {"q": q, "s": s.to(dtype), "z": z, "K": K, "group": group}


def _w4_pack(w, gate_up=False):
    """The package's layout of one weight: made once, kept with the model in place of the checkpoint's."""
    from muxi_race_b200 import pack_w4

    return pack_w4(w["q"], w["s"], w["z"], in_features=w["K"], group_size=w["group"], gate_up=gate_up)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    dtype = DTYPES[case["dtype"]]
    if op in ("norm", "norm_bwd"):
        T, H = case["T"], case["H"]
        s["weight"] = (1 + 0.1 * _randn(gen, H)).to(DTYPES[case["weight"]])
        if op == "norm":
            s["x"] = _randn(gen, T, H).to(dtype)
            s["residual"] = (2 * _randn(gen, T, H)).to(dtype) if case["residual"] else None
        else:
            s["h"] = (2 * _randn(gen, T, H)).to(dtype)
            s["dy"] = _randn(gen, T, H).to(dtype)
            s["dh"] = _randn(gen, T, H).to(dtype) if case["residual"] else None
    elif op in ("route", "route_bwd"):
        s["logits"], s["bias"] = _route_inputs(case, gen)
        if op == "route_bwd":  # the forward's choice, and the gradient of the weights
            s["ids"] = _plain_select(case, s["logits"], s["bias"])
            s["dw"] = _randn(gen, case["T"], case["k"])
    elif op == "linear":
        s["x"] = _randn(gen, case["M"], case["K"]).to(dtype)
        s["w"] = _w4_inputs(gen, (), case["N"], case["K"], case["group"], case["zeros"], dtype)
        if own:
            s["w"] = _w4_pack(s["w"])
    else:
        T, H, I, E, k = (case[n] for n in ("T", "H", "I", "E", "k"))
        s["x"] = _randn(gen, T, H).to(dtype)
        logits = _randn(gen, T, E)
        if case["skew"]:  # expert of popularity rank r is drawn about r^-skew as often
            rank = torch.randperm(E, generator=gen, device="cuda").float() + 1
            logits = logits - case["skew"] * rank.log()
        vals, ids = torch.softmax(logits, -1).topk(k, -1)
        s["ids"] = ids.to(torch.int32).contiguous()
        s["weights"] = (vals / vals.sum(-1, keepdim=True)).contiguous()
        for name, N, K in (("w13", 2 * I, H), ("w2", H, I)):
            s[name] = _w4_inputs(gen, (E,), N, K, case["group"], case["zeros"], dtype)
            if own:
                s[name] = _w4_pack(s[name], gate_up=name == "w13")
    return s


# ------------------------------------------------------------------------------------ the calls
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import muxi_race_b200 as m

    case = s["case"]
    op = case["op"]
    if op == "norm":
        if case["quant"] == "none":
            r = m.add_rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)
            y, h = r if case["residual"] else (r, None)
            return {"y": y, "h": h}
        q, scale, h = m.add_rms_norm_quant(s["x"], s["weight"], s["residual"], eps=EPS, q_dtype=Q_DTYPES[case["quant"]])
        return _quantised(case, q, scale, h)
    if op == "norm_bwd":
        dx, dweight = m.add_rms_norm_backward(s["dy"], s["h"], s["weight"], s["dh"], eps=EPS)
        return {"dx": dx, "dweight": dweight}
    if op in ("route", "route_bwd"):
        how = dict(scoring=case["scoring"], renormalize=case["renorm"], scale=case["scale"])
        if op == "route_bwd":
            return {"dlogits": m.route_topk_backward(s["dw"], s["logits"], s["ids"], **how)}
        w, ids, counts = m.route_topk(s["logits"], case["k"], bias=s["bias"], num_groups=case["groups"],
                                      topk_groups=case["top_groups"], return_counts=True, **how)
        return {"weights": w, "ids": ids, "counts": counts}
    if op == "linear":
        return m.w4_linear(s["x"], s["w"])
    return m.fused_moe_w4(s["x"], s["w13"], s["w2"], s["ids"], s["weights"])


def _quantised(case, q, scale, h):
    """int8 codes as the values they stand for, in the type of the activations; e4m3 values are
    numbers already."""
    if case["quant"] == "int8":
        q = torch.mul(q, scale[:, None], out=torch.empty(q.shape, dtype=DTYPES[case["dtype"]], device=q.device))
    return {"q": q, "scale": scale, "h": h}


def _run_plain(s):
    op = s["case"]["op"]
    if op == "norm":
        return _plain_norm(s)
    if op == "norm_bwd":
        return _plain_norm_bwd(s)
    if op == "route":
        return _plain_route(s)
    if op == "route_bwd":
        return _plain_route_bwd(s)
    if op == "linear":
        return (s["x"].float() @ _plain_w4(s["w"]).T).to(s["x"].dtype)
    return _plain_experts(s)


def _plain_norm(s):
    case, x = s["case"], s["x"]
    h = x.float()
    if case["residual"]:
        h = h + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    h = h.to(x.dtype) if case["residual"] else None
    if case["quant"] == "none":
        return {"y": y.to(x.dtype), "h": h}
    amax = y.abs().amax(-1, keepdim=True)
    v = y * torch.where(amax > 0, Q_MAX[case["quant"]] / amax, 0.0)
    if case["quant"] == "fp8":
        q = v.clamp(-448, 448).to(torch.float8_e4m3fn)
    else:  # nearest, halves away from zero
        q = (v.sign() * (v.abs() + 0.5).floor()).clamp(-127, 127).to(torch.int8)
    return _quantised(case, q, (amax / Q_MAX[case["quant"]]).squeeze(-1), h)


def _plain_norm_bwd(s):
    h, dy, w = s["h"].float(), s["dy"].float(), s["weight"].float()
    r = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    xh, g = h * r, dy * w
    dx = r * (g - xh * (g * xh).mean(-1, keepdim=True))
    if s["dh"] is not None:
        dx = dx + s["dh"].float()
    return {"dx": dx.to(s["dy"].dtype), "dweight": (dy * xh).sum(0).to(s["weight"].dtype)}


def _plain_scores(l, scoring):
    if scoring == "sigmoid":
        return 1 / (1 + torch.exp(-l))
    m = l.amax(-1, keepdim=True)
    e = torch.exp(l - torch.where(m == NEG_INF, 0.0, m))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_select(case, logits, bias):
    """ids [T, k] int32 in descending order, ties to the lowest id, -1 where no expert is left."""
    T, E, n = case["T"], case["E"], case["groups"]
    l = logits.float()
    if bias is None and n == 1:
        c = l  # scores rise with the logits
    else:
        c = _plain_scores(l, case["scoring"])
        c = (c if bias is None else c + bias).masked_fill(l == NEG_INF, NEG_INF)
    if n > 1:
        g = c.view(T, n, E // n).sort(dim=-1, descending=True).values[..., :2].sum(-1)
        best = g.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros(T, n, dtype=torch.bool, device=l.device).scatter_(1, best, True)
        c = c.masked_fill(~keep.repeat_interleave(E // n, 1), NEG_INF)
    v, ids = c.sort(dim=-1, descending=True, stable=True)
    return torch.where(v == NEG_INF, -1, ids)[:, :case["k"]].to(torch.int32).contiguous()


def _plain_route(s):
    case, l = s["case"], s["logits"].float()
    ids = _plain_select(case, s["logits"], s["bias"])
    there = ids >= 0
    at = ids.clamp_min(0).long()
    if case["scoring"] == "softmax" and case["renorm"]:
        w = _plain_scores(l.gather(1, at).masked_fill(~there, NEG_INF), "softmax")
    else:
        w = _plain_scores(l, case["scoring"]).gather(1, at) * there
        if case["renorm"]:
            w = w / w.sum(-1, keepdim=True).clamp_min(1e-20)
    hist = torch.zeros(case["E"], dtype=torch.int32, device=l.device)
    counts = hist.scatter_add_(0, at.reshape(-1), there.reshape(-1).to(torch.int32))
    return {"weights": w * case["scale"], "ids": ids, "counts": counts}


def _plain_route_bwd(s):
    case, l, g = s["case"], s["logits"].float(), s["dw"] * s["case"]["scale"]
    there = s["ids"] >= 0
    at = s["ids"].clamp_min(0).long()
    g = g * there
    if case["scoring"] == "softmax" and case["renorm"]:
        p = _plain_scores(l.gather(1, at).masked_fill(~there, NEG_INF), "softmax")
        d = p * (g - (g * p).sum(-1, keepdim=True))
    else:
        all_p = _plain_scores(l, case["scoring"])
        p = all_p.gather(1, at) * there
        if case["renorm"]:
            den = p.sum(-1, keepdim=True).clamp_min(1e-20)
            g = (g - (g * p).sum(-1, keepdim=True) / den) / den
        if case["scoring"] == "softmax":
            d = g * p
            dl = -all_p * d.sum(-1, keepdim=True)
            return {"dlogits": dl.scatter_add(1, at, d * there).to(s["logits"].dtype)}
        d = g * p * (1 - p)
    return {"dlogits": torch.zeros_like(l).scatter_add(1, at, d * there).to(s["logits"].dtype)}


def _plain_w4(w, index=None):
    """fp32 weights [..., N, K]; with `index` those of the experts it names."""
    q, sc, z = (t if t is None or index is None else t.index_select(0, index) for t in (w["q"], w["s"], w["z"]))
    K, g = w["K"], w["group"]
    v = torch.stack((q & 15, q >> 4), -1).flatten(-2)[..., :K].float()
    z = 8.0 if z is None else z.float().repeat_interleave(g, -1)[..., :K]
    return (v - z) * sc.float().repeat_interleave(g, -1)[..., :K]


def _plain_experts(s):
    case, x = s["case"], s["x"].float()
    T, H, I, k = (case[n] for n in ("T", "H", "I", "k"))
    ids = s["ids"].reshape(-1)
    rows = x.repeat_interleave(k, 0)
    step = max(1, (1 << 28) // (2 * H * I))  # routes whose fp32 weights are held at a time
    y = []
    for r in range(0, T * k, step):
        e = ids[r:r + step]
        gu = torch.bmm(_plain_w4(s["w13"], e), rows[r:r + step, :, None]).squeeze(-1)
        gate, up = gu[:, :I], gu[:, I:]
        a = gate / (1 + torch.exp(-gate)) * up
        y.append(torch.bmm(_plain_w4(s["w2"], e), a[:, :, None]).squeeze(-1))
    y = torch.cat(y).view(T, k, H) * s["weights"][..., None]
    return y.sum(1).to(s["x"].dtype)


# ------------------------------------------------------------------------------------ work
def _w4_bytes(case, N, K):
    return N * K / 2 + N * -(-K // case["group"]) * (3 if case["zeros"] else 2)


def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "f32" else 2
    if op == "norm":
        n = case["T"] * case["H"]
        out = size if case["quant"] == "none" else 1
        b = n * (size + out + (2 * size if case["residual"] else 0)) + case["H"] * (4 if case["weight"] == "f32" else 2)
        return {"bytes": b + (0 if case["quant"] == "none" else 4 * case["T"]), "flops": 5 * n}
    if op == "norm_bwd":
        n = case["T"] * case["H"]
        return {"bytes": n * size * (4 if case["residual"] else 3) + 2 * case["H"] * (4 if case["weight"] == "f32" else 2),
                "flops": 10 * n}
    if op == "route":
        n = case["T"] * case["E"]
        return {"bytes": n * size + 8 * case["T"] * case["k"] + 4 * case["E"], "flops": 4 * n}
    if op == "route_bwd":
        n = case["T"] * case["E"]
        dense = case["scoring"] == "softmax" and not case["renorm"]
        chosen = case["T"] * case["k"]
        return {"bytes": n * size * (2 if dense else 1) + chosen * (8 if dense else 8 + size), "flops": 4 * n}
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": _w4_bytes(case, N, K) + 2 * M * (N + K), "flops": 2 * M * N * K}
    T, H, I, E, k = (case[n] for n in ("T", "H", "I", "E", "k"))
    active = E * (1 - (1 - k / E) ** T)  # experts that some token chose, as expected without skew
    return {"bytes": active * (_w4_bytes(case, 2 * I, H) + _w4_bytes(case, H, I)) + T * (4 * H + 8 * k),
            "flops": 6 * T * k * H * I}


# ------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    global own
    kept, own = own, False  # the checkpoint's form of the weights
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    f = lambda t: t.to(torch.float64)  # noqa: E731
    if op == "norm":
        h = f(s["x"]) + (f(s["residual"]) if case["residual"] else 0)
        y = h / (h.pow(2).mean(1, keepdim=True) + EPS).sqrt() * f(s["weight"])
        h = h if case["residual"] else None
        if case["quant"] == "none":
            return {"y": y, "h": h}
        scale = y.abs().amax(1) / Q_MAX[case["quant"]]
        # int8 is compared as values: how far a code's value is from the unrounded one; e4m3 values
        # stand for y / scale
        return {"q": y / scale[:, None] if case["quant"] == "fp8" else y, "scale": scale, "h": h}
    if op == "norm_bwd":
        h = f(s["h"]).requires_grad_()
        w = f(s["weight"]).requires_grad_()
        y = h / (h.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w
        dx, dw = torch.autograd.grad((y * f(s["dy"])).sum(), (h, w))
        return {"dx": dx + (f(s["dh"]) if case["residual"] else 0), "dweight": dw}
    if op in ("route", "route_bwd"):
        l = f(s["logits"]).requires_grad_()
        p = _route_scores64(l, case["scoring"])
        if op == "route_bwd":
            ids = s["ids"].long()
        else:
            with torch.no_grad():
                c = l if s["bias"] is None and case["groups"] == 1 else p + (0 if s["bias"] is None else f(s["bias"]))
                c = torch.where(l == NEG_INF, NEG_INF, c)
                if case["groups"] > 1:
                    c = c.unflatten(1, (case["groups"], -1))
                    score = c.topk(2, -1).values.sum(-1)
                    order = torch.argsort(score, dim=1, descending=True, stable=True)
                    out = torch.ones_like(score, dtype=torch.bool).scatter(1, order[:, :case["top_groups"]], False)
                    c = c.masked_fill(out[..., None], NEG_INF).flatten(1)
                ids = torch.argsort(c, dim=1, descending=True, stable=True)[:, :case["k"]]
                ids = ids.masked_fill(c.gather(1, ids) == NEG_INF, -1)
        w = torch.where(ids < 0, 0.0, p.gather(1, ids.clamp_min(0)))
        if case["renorm"]:
            w = w / w.sum(1, keepdim=True).clamp_min(1e-290)
        w = w * case["scale"]
        if op == "route_bwd":
            d, = torch.autograd.grad((w * f(s["dw"])).sum(), l)
            return {"dlogits": d}
        counts = torch.bincount(ids[ids >= 0], minlength=case["E"])
        return {"weights": w.detach(), "ids": ids.to(torch.int32), "counts": counts.to(torch.int32)}

    def weights64(w, *at):
        q = w["q"][at]
        v = torch.empty((*q.shape[:-1], 2 * q.shape[-1]), dtype=torch.float64, device=q.device)
        v[..., 0::2], v[..., 1::2] = q % 16, q // 16
        group = torch.arange(w["K"], device=q.device) // w["group"]
        z = 8 if w["z"] is None else f(w["z"][at])[..., group]
        return (v[..., :w["K"]] - z) * f(w["s"][at])[..., group]

    if op == "linear":
        return f(s["x"]) @ weights64(s["w"]).mT
    I = case["I"]
    out = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda")
    for e in s["ids"].unique().tolist():
        t, j = torch.nonzero(s["ids"] == e, as_tuple=True)
        gu = f(s["x"])[t] @ weights64(s["w13"], e).mT
        a = gu[:, :I] * torch.sigmoid(gu[:, :I]) * gu[:, I:]
        out.index_add_(0, t, a @ weights64(s["w2"], e).mT * f(s["weights"])[t, j, None])
    return out
