"""The products with 4-bit weights, their format, and the mixture-of-experts layer that this library's speed is measured on.

A case is one call (a quantisation: there and back) on operands that lie in device memory, as a serving program makes it.  `listed()` holds
the calls that stand for the range, `draw()` makes further ones.  With `own` false `run()` computes the same in elementary torch operations.

4-bit weights: two codes to a byte along k, the even one in the low half; `group` consecutive k of a row share a scale and a zero point
(8 where there are none): w = (code - zero) * scale.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
IDS = {"f32": 0, "f16": 1, "bf16": 3}           # element types as the C ABI numbers them

# what one drawn call may cost: bytes and operations of the largest listed call of its kind
MOST = {"gemm_w4": (2.0e8, 2 * 2048 * 8192 * 4096), "w4_quantize": (4.0e8, 1e9), "moe": (8.5e8, 4e10)}


def _gemm(dtype, m, n, k, group, zeros=False, alpha=1.0, beta=0.0, pad=0):
    """pad: elements between the rows of Q (twice that), the columns of B and of C, as operands inside larger arrays have."""
    return {"op": "gemm_w4", "dtype": dtype, "m": m, "n": n, "k": k, "group": group, "zeros": zeros, "alpha": alpha, "beta": beta, "pad": pad}


def _quantize(w_dtype, dtype, m, k, group, zeros=False, pad=0):
    return {"op": "w4_quantize", "w_dtype": w_dtype, "dtype": dtype, "m": m, "k": k, "group": group, "zeros": zeros, "pad": pad}


def _moe(dtype, tokens, hidden, inner, experts, top_k, group=0, zeros=False, scoring="softmax", renormalize=True, bias=False, beta=0.0, pad=0):
    """group: of 4-bit expert weights; 0: they are in 16 bits."""
    return {"op": "moe", "dtype": dtype, "tokens": tokens, "hidden": hidden, "inner": inner, "experts": experts, "top_k": top_k, "group": group,
            "zeros": zeros, "scoring": scoring, "renormalize": renormalize, "bias": bias, "beta": beta, "pad": pad}


def listed():
    return [
        # one token through a square layer: a call of a few microseconds, where latency counts
        dict(_gemm("f16", 4096, 1, 4096, 128), name="w4_f16_1x4096x4096"),
        # one token through the widest layer: the weights alone are 117 MB
        dict(_gemm("bf16", 28672, 1, 8192, 128, zeros=True), name="w4_bf16_1x28672x8192_zeros"),
        # sixteen sequences decoded together, a long k, small groups
        dict(_gemm("bf16", 4096, 16, 14336, 64), name="w4_bf16_16x4096x14336_g64"),
        # odd in every direction, rows inside larger arrays, added to what is there
        dict(_gemm("f16", 1537, 5, 1003, 32, zeros=True, alpha=0.5, beta=0.5, pad=3), name="w4_f16_5x1537x1003_update"),
        # a batch of 64 sequences
        dict(_gemm("f16", 8192, 64, 8192, 128), name="w4_f16_64x8192x8192"),
        # a prompt: as much arithmetic as weights
        dict(_gemm("bf16", 8192, 2048, 4096, 128), name="w4_bf16_2048x8192x4096"),
        # a small layer with ragged rows to 4 bits and back
        dict(_quantize("f16", "f16", 515, 1000, 32, zeros=True, pad=8), name="quantize_f16_515x1000_zeros"),
        # a large one
        dict(_quantize("bf16", "bf16", 8192, 8192, 128), name="quantize_bf16_8192x8192"),
        # one token through many small experts in 16 bits
        dict(_moe("bf16", 1, 2048, 1024, 64, 8), name="moe_bf16_1_of_64x2048x1024"),
        # eight sequences, the same experts in 4 bits
        dict(_moe("bf16", 8, 2048, 1024, 64, 8, group=128), name="moe_w4_bf16_8_of_64x2048x1024"),
        # odd sizes, sigmoid scores with a bias for the selection, added to what is there
        dict(_moe("f16", 3, 1000, 364, 23, 3, scoring="sigmoid", bias=True, beta=0.5, pad=4), name="moe_f16_3_of_23x1000x364_sigmoid"),
        # a batch of 64 sequences through few large experts: all weights are read
        dict(_moe("bf16", 64, 4096, 2048, 16, 2), name="moe_bf16_64_of_16x4096x2048"),
    ]


def _size(rng, low, high):
    """Spread over the logarithm; half of them as they fall, the others whole multiples of 8, 32 or 128."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    step = rng.choice((1, 1, 1, 8, 32, 128))
    return max(low, v // step * step)


def draw(rng):
    op = rng.choice(("gemm_w4", "gemm_w4", "gemm_w4", "moe", "moe", "w4_quantize"))
    while True:
        dtype, zeros, pad = rng.choice(("f16", "bf16")), rng.random() < 0.4, rng.choice((0, 0, 0, 1, 8))
        group = rng.choice((32, 64, 96, 128, 128, 256))
        if op == "gemm_w4":
            case = _gemm(dtype, _size(rng, 64, 32768), rng.choice((1, 1, _size(rng, 2, 16), _size(rng, 17, 128), _size(rng, 129, 2048))), _size(rng, 64, 16384), group,
                         zeros, rng.choice((1.0, 1.0, 0.5)), rng.choice((0.0, 0.0, 0.5)), pad)
        elif op == "w4_quantize":
            case = _quantize(rng.choice((dtype, "f32")), dtype, _size(rng, 64, 16384), _size(rng, 64, 16384), group, zeros, pad)
        else:
            experts = rng.randint(4, 128)
            case = _moe(dtype, rng.choice((1, _size(rng, 2, 64))), _size(rng, 256, 4096), _size(rng, 128, 4096), experts, rng.randint(1, min(8, experts)),
                        rng.choice((0, group)), zeros, rng.choice(("softmax", "softmax", "sigmoid")), rng.random() < 0.7, rng.random() < 0.3,
                        rng.choice((0.0, 0.0, 0.5)), pad)
            if 6.0 * experts * case["hidden"] * case["inner"] > 4e9:
                continue                         # (what lies in memory, not what is read)
        w, most = work(case), MOST[op]
        if w["bytes"] <= most[0] and w["flops"] <= most[1]:
            return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g, dtype=torch.float32) * scale).to(dtype)


def _columns(rows, cols, pad, dtype, g):
    """`cols` columns of `rows` elements, `rows + pad` apart, of about unit size."""
    return _randn((cols, rows + pad), dtype, g)


def _w4(rows, k, group, zeros, pad, dtype, g, lead=()):
    """Codes [.., rows, bytes], scales and zero points [.., rows, groups] of weights of about 1 / sqrt(k) each."""
    groups = -(-k // group)
    codes = torch.randint(0, 256, lead + (rows, (k + 1) // 2 + pad), device="cuda", generator=g, dtype=torch.uint8)
    scales = ((torch.rand(lead + (rows, groups), device="cuda", generator=g) + 0.5) * (0.2 / math.sqrt(k))).to(dtype)
    z = torch.randint(5, 12, lead + (rows, groups), device="cuda", generator=g, dtype=torch.uint8) if zeros else None
    return codes, scales, z


def prepare(case, seed):
    g, dt, s = _generator(seed), TYPES[case["dtype"]], {"case": case}
    pad = case["pad"]
    if case["op"] == "gemm_w4":
        m, n, k = case["m"], case["n"], case["k"]
        s["q"], s["scales"], s["zeros"] = _w4(m, k, case["group"], case["zeros"], pad, dt, g)
        s["b"] = _columns(k, n, pad, dt, g)
        s["c"] = _columns(m, n, pad, dt, g)
    elif case["op"] == "w4_quantize":
        m, k = case["m"], case["k"]
        groups = -(-k // case["group"])
        s["w"] = _randn((m, k + pad), TYPES[case["w_dtype"]], g, 1 / math.sqrt(k))
        s["q"] = torch.zeros((m, (k + 1) // 2 + pad), device="cuda", dtype=torch.uint8)
        s["scales"] = torch.zeros((m, groups), device="cuda", dtype=dt)
        s["zeros"] = torch.zeros((m, groups), device="cuda", dtype=torch.uint8) if case["zeros"] else None
        s["back"] = torch.zeros((m, k), device="cuda", dtype=dt)
    else:
        t, h, i, e = case["tokens"], case["hidden"], case["inner"], case["experts"]
        s["x"], s["y"] = _columns(h, t, pad, dt, g), _columns(h, t, pad, dt, g)
        s["router"] = _randn((e, h), dt, g, 1.5 / math.sqrt(h))
        s["bias"] = _randn((e,), torch.float32, g, 0.05) if case["bias"] else None
        if case["group"]:
            s["gate_up"] = _w4(2 * i, h, case["group"], case["zeros"], 0, dt, g, (e,))
            s["down"] = _w4(h, i, case["group"], case["zeros"], 0, dt, g, (e,))
        else:
            s["gate_up"] = (_randn((e, 2 * i, h), dt, g, 1 / math.sqrt(h)), None, None)
            s["down"] = (_randn((e, h, i), dt, g, 1 / math.sqrt(i)), None, None)
        s["ids"] = torch.zeros((t, case["top_k"]), device="cuda", dtype=torch.int32)
        s["weights"] = torch.zeros((t, case["top_k"]), device="cuda", dtype=torch.float32)
        if own:
            import gemm_mmbo_amd as G
            s["layer"] = _layer(G, case, s)
            s["workspace"] = torch.empty(G.moe_workspace_bytes(s["layer"], t), device="cuda", dtype=torch.uint8)
    return s


def _layer(G, case, s):
    def matrix(w, k):
        q, scales, zeros = w
        if scales is None:
            return G.moe_matrix(q, k, q.stride(0))
        groups = scales.shape[-1]
        return G.moe_matrix(q, 2 * q.shape[-1], 2 * q.stride(0), scales, groups, scales.stride(0), zeros, groups, scales.stride(0))

    return G.moe_layer(IDS[case["dtype"]], case["hidden"], case["inner"], case["experts"], case["top_k"], s["router"], case["hidden"],
                       matrix(s["gate_up"], case["hidden"]), matrix(s["down"], case["inner"]), group=case["group"], bias=s["bias"],
                       scoring=G.MOE_SIGMOID if case["scoring"] == "sigmoid" else G.MOE_SOFTMAX, renormalize=case["renormalize"])


def _own(s):
    import gemm_mmbo_amd as G
    c = s["case"]
    dt = IDS[c["dtype"]]
    if c["op"] == "gemm_w4":
        m, n, k = c["m"], c["n"], c["k"]
        groups = s["scales"].shape[1]
        G.gemm_w4(dt, m, n, k, c["group"], c["alpha"], s["q"], 2 * s["q"].shape[1], s["scales"], groups, s["zeros"], groups, s["b"], k + c["pad"],
                  c["beta"], s["c"], m + c["pad"])
        return {"c": s["c"][:, :m]}
    if c["op"] == "w4_quantize":
        m, k, groups = c["m"], c["k"], s["scales"].shape[1]
        G.w4_quantize(IDS[c["w_dtype"]], dt, m, k, c["group"], s["w"], k + c["pad"], s["q"], 2 * s["q"].shape[1], s["scales"], groups, s["zeros"], groups)
        G.w4_dequantize(dt, m, k, c["group"], s["q"], 2 * s["q"].shape[1], s["scales"], groups, s["zeros"], groups, s["back"], k)
        return {"w": s["back"], "scales": s["scales"], "zeros": s["zeros"]}
    h = c["hidden"]
    G.moe(s["layer"], c["tokens"], 1.0, s["x"], h + c["pad"], c["beta"], s["y"], h + c["pad"], s["workspace"], s["workspace"].numel(), s["ids"], s["weights"])
    return {"y": s["y"][:, :h], "ids": s["ids"], "weights": s["weights"]}


def _spread(v, group, k):
    """One value for every k from one for every group."""
    return v.repeat_interleave(group, -1)[..., :k]


def _expand(w, k, group):
    """Weights in 32 bits."""
    q, scales, zeros = w
    if scales is None:
        return q.float()
    codes = torch.stack((q & 15, q >> 4), -1).flatten(-2)[..., :k].float()
    z = 8.0 if zeros is None else _spread(zeros.float(), group, k)
    return (codes - z) * _spread(scales.float(), group, k)


def _plain_gemm(s):
    c = s["case"]
    m, k = c["m"], c["k"]
    w = _expand((s["q"], s["scales"], s["zeros"]), k, c["group"])
    y = c["alpha"] * (s["b"][:, :k].float() @ w.t())
    out = s["c"][:, :m]
    out.copy_(y + c["beta"] * out.float() if c["beta"] else y)
    return {"c": out}


def _plain_quantize(s):
    # in 64 bits: codes lie next to the borders of their steps
    c = s["case"]
    m, k, group, dt = c["m"], c["k"], c["group"], TYPES[c["dtype"]]
    groups = -(-k // group)
    w = torch.zeros((m, groups * group), device="cuda", dtype=torch.float64)
    w[:, :k] = s["w"][:, :k]
    w = w.view(m, groups, group)
    if c["zeros"]:
        low, high = w.amin(-1, keepdim=True).clamp(max=0), w.amax(-1, keepdim=True).clamp(min=0)
        scale = ((high - low) / 15).float().to(dt)
        step = torch.where(scale == 0, 1.0, scale.double())
        zero = torch.round(-low / step).clamp(0, 15)
        code = (torch.round(w / step) + zero).clamp(0, 15)
        s["zeros"].copy_(zero.squeeze(-1))
    else:
        scale = (w.abs().amax(-1, keepdim=True) / 7).float().to(dt)
        step = torch.where(scale == 0, 1.0, scale.double())
        zero = 8.0
        code = (torch.round(w / step) + 8).clamp(0, 15)
    s["scales"].copy_(scale.squeeze(-1))
    s["back"].copy_(((code - zero) * scale.double()).float().to(dt).view(m, -1)[:, :k])
    return {"w": s["back"], "scales": s["scales"], "zeros": s["zeros"]}


def _route(s):
    """(expert ids, weights) of each token; in 64 bits, so that the selection does not hang on the order of a sum."""
    c = s["case"]
    logits = s["x"][:, :c["hidden"]].double() @ s["router"].double().t()
    if c["scoring"] == "sigmoid":
        score = 1 / (1 + torch.exp(-logits))
    else:
        score = torch.exp(logits - logits.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    key = logits if s["bias"] is None else score + s["bias"].double()
    ids = torch.sort(key, dim=1, descending=True, stable=True)[1][:, :c["top_k"]]
    weights = score.gather(1, ids)
    if c["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    return ids, weights


def _plain_moe(s):
    c = s["case"]
    t, h, i, e, top = c["tokens"], c["hidden"], c["inner"], c["experts"], c["top_k"]
    ids, weights = _route(s)
    x = s["x"][:, :h].float()
    few = t * top <= e
    chosen = ids.flatten() if few else slice(None)          # few tokens: the experts that they take, otherwise all of them
    def pick(w):
        return tuple(v if v is None else v[chosen] for v in w)
    right = x.repeat_interleave(top, 0).unsqueeze(-1) if few else x.t().contiguous()
    gate_up = torch.matmul(_expand(pick(s["gate_up"]), h, c["group"]), right)
    gate, up = gate_up[:, :i], gate_up[:, i:]
    inner = gate / (1 + torch.exp(-gate)) * up
    out = torch.matmul(_expand(pick(s["down"]), i, c["group"]), inner)
    if few:
        y = (out.view(t, top, h) * weights.float().unsqueeze(-1)).sum(1)
    else:
        share = torch.zeros((t, e), device="cuda").scatter_(1, ids, weights.float())
        y = (out * share.t().unsqueeze(1)).sum(0).t()
    to = s["y"][:, :h]
    to.copy_(y + c["beta"] * to.float() if c["beta"] else y)
    s["ids"].copy_(ids)
    s["weights"].copy_(weights)
    return {"y": to, "ids": s["ids"], "weights": s["weights"]}


def run(state):
    if own:
        return _own(state)
    return {"gemm_w4": _plain_gemm, "w4_quantize": _plain_quantize, "moe": _plain_moe}[state["case"]["op"]](state)


def _active(case):
    """How many experts a batch is expected to reach."""
    e = case["experts"]
    return e * (1 - (1 - case["top_k"] / e) ** case["tokens"])


def work(case):
    def w4_bytes(rows, k):
        return rows * k / 2 + rows * -(-k // case["group"]) * (3 if case["zeros"] else 2)

    if case["op"] == "gemm_w4":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": w4_bytes(m, k) + 2 * n * k + 2 * m * n * (2 if case["beta"] else 1), "flops": 2 * m * n * k}
    if case["op"] == "w4_quantize":
        m, k = case["m"], case["k"]
        return {"bytes": m * k * (4 if case["w_dtype"] == "f32" else 2) + 2 * w4_bytes(m, k) + 2 * m * k, "flops": 6 * m * k}
    t, h, i, e = case["tokens"], case["hidden"], case["inner"], case["experts"]
    weights = w4_bytes(2 * i, h) + w4_bytes(h, i) if case["group"] else 6 * h * i
    return {"bytes": _active(case) * weights + 2 * e * h + 2 * t * h * (3 if case["beta"] else 2), "flops": 2 * t * h * (e + 3 * case["top_k"] * i)}


# ---- from the definitions, in 64 bits, row by row and expert by expert

def _exact_weights(q, scales, zeros, k, group):
    if scales is None:
        return q.double()
    l = torch.arange(k, device="cuda")
    code = torch.bitwise_right_shift(q[..., l // 2].to(torch.int32), 4 * (l % 2).to(torch.int32)) & 15
    z = zeros.double()[..., l // group] if zeros is not None else 8
    return (code - z) * scales.double()[..., l // group]


def _exact_gemm(case, s):
    y = torch.empty((case["n"], case["m"]), device="cuda", dtype=torch.float64)
    b = s["b"][:, :case["k"]].double()
    for r in range(0, case["m"], 2048):                     # (some rows at a time: memory)
        part = slice(r, r + 2048)
        w = _exact_weights(s["q"][part], s["scales"][part], None if s["zeros"] is None else s["zeros"][part], case["k"], case["group"])
        y[:, part] = (w @ b.t()).t()
    return {"c": case["alpha"] * y + (case["beta"] * s["c"][:, :case["m"]].double() if case["beta"] else 0)}


def _exact_quantize(case, s):
    m, k, group, dt = case["m"], case["k"], case["group"], TYPES[case["dtype"]]
    w = s["w"][:, :k].double()
    groups = -(-k // group)
    back, scales = torch.empty((m, k), device="cuda", dtype=torch.float64), torch.empty((m, groups), device="cuda", dtype=torch.float64)
    for g in range(groups):
        v = w[:, g * group:(g + 1) * group]
        low, high = v.min(1).values, v.max(1).values
        if case["zeros"]:
            span = (torch.maximum(high, torch.zeros_like(high)) - torch.minimum(low, torch.zeros_like(low))) / 15
        else:
            span = torch.maximum(high, -low) / 7
        # the format holds the scale in the weights' type: that rounding is part of its definition
        scale = span.to(torch.float32).to(dt).double()
        scales[:, g] = scale
        safe = scale.masked_fill(scale == 0, 1)[:, None]
        if case["zeros"]:
            zero = torch.clamp(torch.round(torch.clamp(-low, min=0)[:, None] / safe), 0, 15)
            level = torch.clamp(torch.round(v / safe), -zero, 15 - zero)
        else:
            level = torch.clamp(torch.round(v / safe), -8, 7)
        back[:, g * group:(g + 1) * group] = level * scale[:, None]
    return {"w": back, "scales": scales, "zeros": None}


def _exact_moe(case, s):
    t, h, i, top = case["tokens"], case["hidden"], case["inner"], case["top_k"]
    x = s["x"][:, :h].double()
    y = case["beta"] * s["y"][:, :h].double() if case["beta"] else torch.zeros((t, h), device="cuda", dtype=torch.float64)
    logits = (s["router"].double() @ x.t()).t()
    score = torch.sigmoid(logits) if case["scoring"] == "sigmoid" else torch.softmax(logits, 1)
    key = (logits if s["bias"] is None else score + s["bias"].double()).tolist()
    ids = torch.tensor([sorted(range(len(r)), key=lambda e, r=r: (-r[e], e))[:top] for r in key], device="cuda")
    weights = torch.stack([score[a][ids[a]] for a in range(t)])
    if case["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    for e in sorted(set(ids.flatten().tolist())):
        a, slot = torch.nonzero(ids == e, as_tuple=True)
        w = [_exact_weights(*(v if v is None else v[e] for v in s[name]), k, case["group"]) for name, k in (("gate_up", h), ("down", i))]
        g, u = x[a] @ w[0][:i].t(), x[a] @ w[0][i:].t()
        y[a] += weights[a, slot][:, None] * ((g * torch.sigmoid(g) * u) @ w[1].t())
    return {"y": y, "ids": ids, "weights": weights}


def exact(case, seed):
    s = prepare(case, seed)
    return {"gemm_w4": _exact_gemm, "w4_quantize": _exact_quantize, "moe": _exact_moe}[case["op"]](case, s)
