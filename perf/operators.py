"""Cases for the expert half of a block: MXFP4 quantisation and products, routing to experts, and the experts' two products.

Plain values describe a case; ``prepare`` makes what a serving program holds before the call (activations, MXFP4 weights as a
checkpoint stores them, the router's answer), ``run`` is one call, in plain torch operations or through ``tritonllm_amd``.
MXFP4: 32 values share a scale byte s; a value is FP4[code] * 2^(s - 127), two codes to a byte, the low nibble first."""
from __future__ import annotations

import math

import torch

own = False

FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
ALPHA, LIMIT = 1.702, 7.0
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one token's normalised activations before a product with a 4-bit weight: latency alone
        {"name": "quantize_token", "op": "quantize", "rows": 1, "k": 2880, "type": "bf16"},
        # the QKV weights of eight layers, converted from fp32
        {"name": "quantize_weight", "op": "quantize", "rows": 40960, "k": 2880, "type": "f32"},
        # the attention out-projection of one token
        {"name": "linear_token", "op": "linear", "rows": 1, "n": 2880, "k": 4096, "acts": "bf16"},
        # the QKV projection of a decode batch
        {"name": "linear_batch", "op": "linear", "rows": 65, "n": 5120, "k": 2880, "acts": "bf16"},
        # the QKV projection of a prompt with activations quantised on the way in
        {"name": "linear_prompt_4bit", "op": "linear", "rows": 2048, "n": 5120, "k": 2880, "acts": "mxfp4"},
        # the router of a decode batch: the best four of 32 experts
        {"name": "route_batch", "op": "route", "tokens": 8, "experts": 32, "top": 4, "score": "softmax", "groups": 1, "kept": 1, "balanced": False},
        # a long prompt through a router with sigmoid scores, a bias for balance and groups
        {"name": "route_prompt", "op": "route", "tokens": 8191, "experts": 256, "top": 8, "score": "sigmoid", "groups": 8, "kept": 4, "balanced": True},
        # the experts' first product: a single token, a decode batch, a prompt
        {"name": "mlp1_token", "op": "mlp1", "tokens": 1, "experts": 32, "top": 4, "hidden": 2880, "inner": 2880},
        {"name": "mlp1_batch", "op": "mlp1", "tokens": 33, "experts": 32, "top": 4, "hidden": 2880, "inner": 2880},
        {"name": "mlp1_prompt", "op": "mlp1", "tokens": 2048, "experts": 32, "top": 4, "hidden": 2880, "inner": 2880},
        # the experts' second product with the weighted sum and the residual: a decode batch, a prompt
        {"name": "mlp2_batch", "op": "mlp2", "tokens": 8, "experts": 32, "top": 4, "hidden": 2880, "inner": 2880},
        {"name": "mlp2_prompt", "op": "mlp2", "tokens": 2000, "experts": 32, "top": 4, "hidden": 2880, "inner": 2880},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
    """A width of whole blocks: one of the repository's, or an odd number of blocks."""
    if rng.random() < 0.3:
        return rng.choice([w for w in (64, 512, 1024, 2048, 2880, 4096, 5120) if lo <= w <= hi])
    return 32 * (_between(rng, lo // 32, hi // 32 - 1) | 1)


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "route", "mlp1", "mlp1", "mlp2", "mlp2"])
    if op == "quantize":
        return {"op": op, "rows": _between(rng, 1, 40000) | 1, "k": _width(rng, 32, 2880), "type": rng.choice(["bf16", "f16", "f32"])}
    if op == "linear":
        return {"op": op, "rows": _between(rng, 1, 2000) | 1, "n": rng.choice([_width(rng, 64, 5120), _between(rng, 16, 5100) | 1]), "k": _width(rng, 64, 2880),
                "acts": rng.choice(["bf16", "mxfp4"])}
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        score = "sigmoid" if groups > 1 else rng.choice(["softmax", "sigmoid"])
        experts = groups * rng.randint(4, 256 // groups)
        kept = rng.randint(max(1, groups // 2), groups)
        return {"op": op, "tokens": _between(rng, 1, 8000) | 1, "experts": experts, "top": rng.randint(1, min(8, experts // groups * kept)),
                "score": score, "groups": groups, "kept": kept, "balanced": score == "sigmoid" and rng.random() < 0.7}
    experts = rng.choice([4, 8, 17, 32, 64])
    hidden, inner = _width(rng, 64, 2880), _width(rng, 64, 2880)
    at_most = max(1, int(2000 * 4 * 2880 * 2880 / (hidden * inner)))
    top = rng.randint(1, 4)
    return {"op": op, "tokens": _between(rng, 1, min(2001, at_most)) | 1, "experts": experts, "top": top, "hidden": hidden, "inner": inner}


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _mxfp4(g, *shape):
    """Random MXFP4 weights as a quantised normal distribution has them: blocks [..., G, 16], scales [..., G]."""
    levels = torch.tensor(FP4, device="cuda")
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    z = 2.2 * math.sqrt(2) * torch.erfinv((torch.arange(256, device="cuda") + 0.5) / 128 - 1)
    code = (torch.bucketize(z.abs(), edges) + 8 * (z < 0)).to(torch.uint8)      # 256 equally likely values of the distribution
    assert len(levels) == 16
    *rows, k = shape
    pick = torch.randint(0, 256, (*rows, k // 32, 32), generator=g, device="cuda", dtype=torch.uint8)
    codes = code[pick.int()]
    del pick
    blocks = (codes[..., 0::2] | (codes[..., 1::2] << 4)).contiguous()
    scales = torch.randint(118, 122, (*rows, k // 32), generator=g, device="cuda", dtype=torch.uint8)
    return blocks, scales


def _routing(g, tokens, experts, top):
    """What the router answered for uneven experts: chosen experts and weights by token, pairs in the order of their experts, and
    each expert's first place in that order."""
    logits = torch.randn(tokens, experts, generator=g, device="cuda") + 0.5 * torch.randn(experts, generator=g, device="cuda")
    value, chosen = torch.sort(logits, dim=1, descending=True, stable=True)
    chosen = chosen[:, :top].int().contiguous()
    weights = torch.softmax(value[:, :top], dim=1).contiguous()
    flat = chosen.reshape(-1).long()
    order = torch.sort(flat, stable=True).indices.int()
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.cumsum(torch.bincount(flat, minlength=experts), 0)
    return chosen, weights, order, offsets


def prepare(case, seed):
    g = _generator(seed)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s = dict(case)
    if case["op"] == "quantize":
        x = rand(case["rows"], case["k"])
        x *= torch.exp(0.7 * rand(case["k"]))          # channels of unlike size, as activations and weights have
        s["x"] = x.to(TYPES[case["type"]])
    elif case["op"] == "linear":
        s["x"] = rand(case["rows"], case["k"]).bfloat16()
        s["w"], s["ws"] = _mxfp4(g, case["n"], case["k"])
        s["bias"] = rand(case["n"]).bfloat16()
    elif case["op"] == "route":
        s["logits"] = (1.5 * rand(case["tokens"], case["experts"])).bfloat16()
        s["bias"] = 0.1 * rand(case["experts"]) if case["balanced"] else None
    else:
        k, n = (case["hidden"], 2 * case["inner"]) if case["op"] == "mlp1" else (case["inner"], case["hidden"])
        s["chosen"], s["weights"], s["order"], s["offsets"] = _routing(g, case["tokens"], case["experts"], case["top"])
        s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())           # rows of the busiest expert
        s["w"], s["ws"] = _mxfp4(g, case["experts"], n, k)
        s["bias"] = rand(case["experts"], n).bfloat16()
        if case["op"] == "mlp1":
            s["x"] = rand(case["tokens"], k).bfloat16()
        else:
            s["x"] = rand(case["tokens"] * case["top"], k).bfloat16()
            s["residual"] = rand(case["tokens"], n).bfloat16()
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def _values(blocks, scales):
    """MXFP4 -> fp32, [..., G * 32]."""
    codes = torch.stack((blocks & 15, blocks >> 4), dim=-1).flatten(-2)
    v = torch.tensor(FP4, device=blocks.device)[codes.int()]
    v *= torch.exp2(scales.float() - 127)[..., None]
    return v.flatten(-2)


def _quantized(x):
    """Values and scale bytes of x in MXFP4: a power of two for each 32 values, the values to the nearest, ties to even."""
    v = x.float().unflatten(-1, (-1, 32))
    top = v.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top).exponent - 3).clamp(-127, 127)
    e = torch.where(top > 0, e, -127)
    a = v * torch.exp2(-e.float())
    m = a.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    q = torch.copysign((torch.round(m / step) * step).clamp(max=6), a)
    return (q * torch.exp2(e.float())).flatten(-2), (e + 127).to(torch.uint8).squeeze(-1)


def _route(s):
    logits = s["logits"].float()
    tokens, experts = logits.shape
    if s["score"] == "softmax":
        score = torch.exp(logits - logits.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-logits))
    choice = logits if s["bias"] is None else score + s["bias"]
    if s["groups"] > 1:
        by_group = choice.unflatten(1, (s["groups"], -1))
        best = torch.sort(by_group, dim=2, descending=True).values
        if s["bias"] is None:
            value = 1 / (1 + torch.exp(-best[..., 0])) + 1 / (1 + torch.exp(-best[..., 1]))
        else:
            value = best[..., 0] + best[..., 1]
        kept = torch.sort(value, dim=1, descending=True, stable=True).indices[:, : s["kept"]]
        mask = torch.zeros_like(value, dtype=torch.bool).scatter_(1, kept, True)
        choice = by_group.masked_fill(~mask[..., None], -math.inf).flatten(1)
    chosen = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, : s["top"]]
    weights = torch.gather(score, 1, chosen)
    weights = weights / weights.sum(1, keepdim=True)
    flat = chosen.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    first = torch.cumsum((flat[:, None] == torch.arange(experts, device=flat.device)).sum(0), 0)
    return {"experts": chosen.int(), "weights": weights, "order": order.int(), "offsets": torch.cat((first.new_zeros(1), first)).int()}


def _by_expert(s, rows):
    """rows [P, K], in the order of their experts, times each one's expert's weight, plus its bias: [P, N] in fp32."""
    place = torch.arange(rows.shape[0], device=rows.device)
    expert = torch.searchsorted(s["offsets"][1:].contiguous(), place.int(), right=True)
    if rows.shape[0] <= s["experts"]:                      # fewer rows than experts: their experts' weights alone
        y = torch.bmm(_values(s["w"][expert], s["ws"][expert]), rows[:, :, None])[..., 0]
    else:
        at = place - s["offsets"][expert]
        filled = rows.new_zeros(s["experts"], rows.shape[1], s["most"])
        filled[expert, :, at] = rows
        y = torch.bmm(_values(s["w"], s["ws"]), filled)[expert, :, at]
    return y + s["bias"].float()[expert]


def _swiglu(v):
    gate, linear = v[:, 0::2].clamp(max=LIMIT), v[:, 1::2].clamp(-LIMIT, LIMIT)
    return gate / (1 + torch.exp(-ALPHA * gate)) * (linear + 1)


def _plain(s):
    op = s["op"]
    if op == "quantize":
        values, scales = _quantized(s["x"])
        return {"values": values.bfloat16(), "scales": scales}
    if op == "linear":
        x = _quantized(s["x"])[0] if s["acts"] == "mxfp4" else s["x"].float()
        return (x @ _values(s["w"], s["ws"]).t() + s["bias"].float()).bfloat16()
    if op == "route":
        return _route(s)
    if op == "mlp1":
        return _swiglu(_by_expert(s, s["x"].float()[s["order"] // s["top"]])).bfloat16()
    y = _by_expert(s, s["x"].float())
    pair = torch.empty_like(y)
    pair[s["order"].long()] = y
    y = (pair.unflatten(0, (-1, s["top"])) * s["weights"][..., None]).sum(1)
    return (y + s["residual"].float()).bfloat16()


def run(s):
    if not own:
        return _plain(s)
    import tritonllm_amd as T

    op = s["op"]
    if op == "quantize":
        blocks, scales = T.mxfp4_quantize(s["x"])
        return {"values": T.mxfp4_dequant(blocks, scales), "scales": scales}
    if op == "linear":
        if s["acts"] == "mxfp4":
            blocks, scales = T.mxfp4_quantize(s["x"])
            return T.mxfp4_linear(blocks, s["w"], s["ws"], s["bias"], x_scales=scales)
        return T.mxfp4_linear(s["x"], s["w"], s["ws"], s["bias"])
    if op == "route":
        r = T.moe_route(s["logits"], s["top"], score=s["score"], bias=s["bias"], n_groups=s["groups"], topk_groups=s["kept"])
        return {"experts": r.experts, "weights": r.weights, "order": r.order, "offsets": r.offsets}
    routing = T.MoeRouting(s["chosen"], s["weights"], s["order"], s["offsets"])
    if op == "mlp1":
        return T.moe_mlp1(s["x"], routing, s["w"], s["ws"], s["bias"], alpha=ALPHA, limit=LIMIT)
    return T.moe_mlp2(s["x"], routing, s["w"], s["ws"], s["bias"], residual=s["residual"])


def work(case):
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["k"]
        return {"bytes": n * (2 + {"bf16": 2, "f16": 2, "f32": 4}[case["type"]]) + n // 32, "flops": 0}
    if op == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": 2 * rows * (n + k) + n * k * 17 // 32 + 2 * n, "flops": 2 * rows * n * k}
    if op == "route":
        return {"bytes": 2 * case["tokens"] * case["experts"] + 12 * case["tokens"] * case["top"] + 4 * case["experts"], "flops": 0}
    pairs = case["tokens"] * case["top"]
    touched = case["experts"] * (1 - (1 - case["top"] / case["experts"]) ** case["tokens"])     # experts that some token chose, on average
    weight = touched * (2 if op == "mlp1" else 1) * case["hidden"] * case["inner"] * 17 / 32
    rows = 2 * case["tokens"] * case["hidden"] + 2 * pairs * case["inner"]
    rows = rows if op == "mlp1" else rows + 2 * case["tokens"] * case["hidden"]
    return {"bytes": weight + rows + 8 * pairs, "flops": (4 if op == "mlp1" else 2) * pairs * case["hidden"] * case["inner"]}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------
def _weight64(blocks, scales):
    out = torch.empty(*blocks.shape[:-1], 32, dtype=torch.float64, device=blocks.device)
    table = torch.tensor(FP4, dtype=torch.float64, device=blocks.device)
    out[..., 0::2] = table[(blocks % 16).int()]
    out[..., 1::2] = table[(blocks // 16).int()]
    return torch.ldexp(out, (scales.int() - 127)[..., None]).reshape(*blocks.shape[:-2], -1)


def _quantized64(x):
    """To the nearest of the eight magnitudes by comparison with the midpoints; a midpoint goes to the even code."""
    v = x.double().reshape(*x.shape[:-1], -1, 32)
    top = v.abs().max(-1, keepdim=True).values
    e = torch.where(top > 0, torch.floor(torch.log2(top)), -125.0).clamp(-125, 129) - 2
    a = (v / 2.0**e).abs()
    magnitude = torch.zeros_like(a)
    levels = FP4[:8]
    for i in range(1, 8):
        middle = (levels[i - 1] + levels[i]) / 2
        magnitude[(a > middle) | ((a == middle) & (i % 2 == 0))] = levels[i]
    return (torch.sign(v) * magnitude * 2.0**e).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return {"values": _quantized64(s["x"]), "scales": None}
    if op == "linear":
        x = _quantized64(s["x"]) if case["acts"] == "mxfp4" else s["x"].double()
        return torch.addmm(s["bias"].double(), x, _weight64(s["w"], s["ws"]).t())
    if op == "route":
        z = s["logits"].double()
        score = torch.softmax(z, 1) if case["score"] == "softmax" else torch.sigmoid(z)
        choice = score if s["bias"] is None else score + s["bias"].double()
        if case["groups"] > 1:
            members = choice.view(len(z), case["groups"], -1)
            value = members.topk(2, dim=2).values.sum(2)
            rank = torch.argsort(torch.argsort(value, dim=1, descending=True, stable=True), dim=1)
            choice = torch.where((rank < case["kept"])[..., None], members, -1e300).reshape(z.shape)
        best = torch.argsort(choice, dim=1, descending=True, stable=True)[:, : case["top"]]
        weights = score.gather(1, best)
        return {"experts": None, "weights": weights / weights.sum(1, keepdim=True), "order": None, "offsets": None}
    pairs = case["tokens"] * case["top"]
    n = s["w"].shape[1]
    rows = s["x"].double()
    if op == "mlp1":
        rows = rows[torch.div(s["order"], case["top"], rounding_mode="floor")]
    y = torch.empty(pairs, n, dtype=torch.float64, device=rows.device)
    first = s["offsets"].tolist()
    for e in range(case["experts"]):
        lo, hi = first[e], first[e + 1]
        if hi > lo:
            y[lo:hi] = rows[lo:hi] @ _weight64(s["w"][e], s["ws"][e]).t() + s["bias"][e].double()
    if op == "mlp1":
        gate, linear = torch.clamp(y[:, ::2], max=LIMIT), torch.clamp(y[:, 1::2], -LIMIT, LIMIT)
        return gate * torch.sigmoid(ALPHA * gate) * (linear + 1)
    out = s["residual"].double()
    weight = s["weights"].double().reshape(-1)[s["order"].long()]
    out.index_add_(0, torch.div(s["order"], case["top"], rounding_mode="floor").long(), y * weight[:, None])
    return out
