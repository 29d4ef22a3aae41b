"""Cases for a KV cache held in 4 bits: quantising keys and values as they are written, reading them back, and attention over the cache as it
lies, of one new token per sequence and of several.

Plain values describe a case; ``prepare`` makes what a serving program holds before the call (new keys and values, queries, a cache with a
past in it), ``run`` is one call, in plain torch operations or through ``tritonllm_amd``.
The cache is MXFP4: the 32 values of a block share a scale byte s; a value is FP4[code] * 2^(s - 127), two codes to a byte, the low nibble
first. ``[batch, slots, KV heads, head size / 32]`` blocks of 16 bytes and as many scale bytes, for keys and for values, with a head's slots
next to each other in memory."""
from __future__ import annotations

import math

import torch

own = False

FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HEADS = {"kv_heads": 8, "group": 8, "sinks": True, "window": 0, "ragged": False}          # 64 query heads of 64


def listed():
    return [
        # the keys and values of a decode step's eight tokens: latency alone
        {"name": "write_token", "op": "write", "batch": 8, "tokens": 1, "first": 777, "slots": 1024, "kv_heads": 8, "dim": 64, "type": "bf16", "padded": False},
        # three prompts of unlike length as one padded batch, from fp32 activations: what lies behind a sequence's end stays as it was
        {"name": "write_padded", "op": "write", "batch": 3, "tokens": 333, "first": 0, "slots": 1000, "kv_heads": 8, "dim": 64, "type": "f32", "padded": True},
        # a long prompt
        {"name": "write_prompt", "op": "write", "batch": 1, "tokens": 8192, "first": 0, "slots": 8192, "kv_heads": 8, "dim": 64, "type": "bf16", "padded": False},
        # a conversation read back for a consumer of bf16 keys and values
        {"name": "read_prefix", "op": "read", "batch": 1, "tokens": 1500, "first": 0, "slots": 4096, "kv_heads": 8, "dim": 64},
        # eight of them at the original context length
        {"name": "read_batch", "op": "read", "batch": 8, "tokens": 4096, "first": 0, "slots": 4096, "kv_heads": 8, "dim": 64},
        # one user, early in a conversation, in a cache with room for more: latency
        {"name": "decode_1x300", "op": "decode", "batch": 1, "queries": 1, "keys": 300, "slots": 4096, **HEADS},
        # the batch this repository's benchmark is quoted at, at the original context length
        {"name": "decode_8x4096", "op": "decode", "batch": 8, "queries": 1, "keys": 4096, "slots": 4096, **HEADS},
        # long contexts: the cache is all there is to read
        {"name": "decode_8x32768", "op": "decode", "batch": 8, "queries": 1, "keys": 32768, "slots": 32768, **HEADS},
        # a continuous batch of odd size whose sequences are of unlike length
        {"name": "decode_49_ragged", "op": "decode", "batch": 49, "queries": 1, "keys": 2048, "slots": 2048, **{**HEADS, "ragged": True}},
        # four drafted tokens per sequence, to be verified in one pass
        {"name": "drafts_8x4_after_4092", "op": "attention", "batch": 8, "queries": 4, "keys": 4096, "slots": 4608, **HEADS},
        # a chat's next turn: few new tokens behind a conversation
        {"name": "turn_97_after_1500", "op": "attention", "batch": 1, "queries": 97, "keys": 1597, "slots": 4096, **HEADS},
        # one prompt of the ordinary benchmark length
        {"name": "prompt_2048", "op": "attention", "batch": 1, "queries": 2048, "keys": 2048, "slots": 2048, **HEADS},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "decode", "decode", "attention", "attention", "attention"])
    if op in ("write", "read"):
        heads, dim = rng.choice([1, 2, 3, 4, 8, 8, 16]), rng.choice([32, 64, 64, 96, 128, 256])
        batch = _between(rng, 1, 49)
        tokens = _between(rng, 1, max(1, (1 if op == "write" else 4) * 8192 * 512 // (batch * heads * dim)))
        first = rng.choice([0, rng.randint(1, 500)])
        case = {"op": op, "batch": batch, "tokens": tokens, "first": first, "slots": first + tokens + rng.randint(0, 100), "kv_heads": heads, "dim": dim}
        return {**case, "type": rng.choice(["bf16", "f16", "f32"]), "padded": rng.random() < 0.4} if op == "write" else case
    heads, group = rng.choice([(8, 8), (8, 8), (8, 8), (1, 8), (2, 16), (4, 4), (8, 1), (5, 3), (16, 2), (2, 7), (1, 12)])
    case = {"op": op, "kv_heads": heads, "group": group, "sinks": rng.random() < 0.7, "window": rng.choice([0, 0, 128, rng.randint(1, 700)]), "ragged": rng.random() < 0.5}
    if op == "decode":
        queries, batch = 1, _between(rng, 1, 64)
        keys = _between(rng, 1, min(32768, 8 * 32768 * 8 // (batch * heads)))
    else:
        queries = _between(rng, 2, rng.choice([16, 1500]))
        batch = _between(rng, 1, 16 if queries <= 16 else 4)
        most = min(16384, 2048 * 2048 * 64 // (2 * batch * queries * heads * group))
        if queries > most:
            queries = batch = 2
            most = 8192
        keys = _between(rng, queries, most)
    return {**case, "batch": batch, "queries": queries, "keys": keys, "slots": keys + rng.choice([0, 0, rng.randint(1, 3000)])}


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _mxfp4(g, batch, slots, heads, dim):
    """Blocks and scale bytes of normally distributed values, by slots outside and by heads in memory."""
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    z = 2.2 * math.sqrt(2) * torch.erfinv((torch.arange(256, device="cuda") + 0.5) / 128 - 1)
    code = (torch.bucketize(z.abs(), edges) + 8 * (z < 0)).to(torch.uint8)      # 256 equally likely values of the distribution
    two = torch.randint(0, 256, (2, batch, heads, slots, dim // 32, 16), generator=g, device="cuda", dtype=torch.uint8).int()
    blocks = code[two[0]] | (code[two[1]] << 4)
    scales = torch.randint(124, 127, (batch, heads, slots, dim // 32), generator=g, device="cuda", dtype=torch.uint8)
    return blocks.transpose(1, 2), scales.transpose(1, 2)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s = dict(case)
    batch, heads, slots = case["batch"], case["kv_heads"], case["slots"]
    dim = case.get("dim", 64)
    s["cache"] = (*_mxfp4(g, batch, slots, heads, dim), *_mxfp4(g, batch, slots, heads, dim))
    if case["op"] == "write":
        channels = torch.exp(0.5 * rand(2, heads, dim))                 # channels of unlike size, as keys have
        shape = (batch, case["tokens"], heads, dim)
        s["k"], s["v"] = ((rand(*shape) * c).to(TYPES[case["type"]]) for c in channels)
        s["offset"] = torch.full((1,), case["first"], dtype=torch.int64, device="cuda")
        s["lengths"] = torch.randint(0, case["tokens"] + 1, (batch,), generator=g, device="cuda") if case["padded"] else None
    elif case["op"] != "read":
        s["q"] = (2 * rand(batch, case["queries"], heads, case["group"], 64)).bfloat16()
        s["sink"] = rand(heads * case["group"]).bfloat16() if case["sinks"] else None
        last = case["keys"] - case["queries"]                           # the first query's position, in the longest sequence
        s["start"] = torch.full((1,), last, dtype=torch.int64, device="cuda")
        if case["ragged"]:
            s["start"] = torch.randint(0, last + 1, (batch,), generator=g, device="cuda")
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def _values(blocks, scales):
    """MXFP4 -> fp32, [..., G * 32]."""
    codes = torch.stack((blocks & 15, blocks >> 4), dim=-1).flatten(-2)
    v = torch.tensor(FP4, device=blocks.device)[codes.int()]
    return (v * torch.exp2(scales.float() - 127)[..., None]).flatten(-2)


def _quantized(x):
    """The values of x in MXFP4: a power of two for each 32, the values to the nearest, ties to even."""
    v = x.float().unflatten(-1, (-1, 32))
    top = v.abs().amax(-1, keepdim=True)
    e = torch.where(top > 0, (torch.frexp(top).exponent - 3).clamp(-127, 127), -127)
    a = v * torch.exp2(-e.float())
    m = a.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    q = torch.copysign((torch.round(m / step) * step).clamp(max=6), a)
    return (q * torch.exp2(e.float())).flatten(-2)


def _stored(s, blocks, scales, new):
    """What the slots written to hold afterwards."""
    span = slice(s["first"], s["first"] + s["tokens"])
    old, new = _values(blocks[:, span], scales[:, span]), _quantized(new)
    if s["lengths"] is not None:
        written = torch.arange(s["tokens"], device=new.device) < s["lengths"][:, None]
        new = torch.where(written[..., None, None], new, old)
    return new.bfloat16()


def _plain(s):
    kb, ks, vb, vs = s["cache"]
    if s["op"] == "write":
        return {"k": _stored(s, kb, ks, s["k"]), "v": _stored(s, vb, vs, s["v"])}
    if s["op"] == "read":
        span = slice(s["first"], s["first"] + s["tokens"])
        return {"k": _values(kb[:, span], ks[:, span]).bfloat16(), "v": _values(vb[:, span], vs[:, span]).bfloat16()}
    # a KV head's queries are rows of one product with its keys
    n, t, b, h, g = s["keys"], s["queries"], s["batch"], s["kv_heads"], s["group"]
    k = _values(kb[:, :n], ks[:, :n]).permute(0, 2, 3, 1).contiguous()          # [b, h, 64, n]
    v = _values(vb[:, :n], vs[:, :n]).transpose(1, 2).contiguous()              # [b, h, n, 64]
    q = s["q"].float().transpose(1, 2).reshape(b, h, t * g, 64)
    z = (torch.matmul(q, k) * 0.125).view(b, h, t, g, n)
    key = torch.arange(n, device=z.device)
    at = s["start"].view(-1, 1) + torch.arange(t, device=z.device)              # [1 or b, t]
    seen = key <= at[..., None]
    if s["window"]:
        seen = seen & (key > at[..., None] - s["window"])
    z = z.masked_fill(~seen[:, None, :, None, :], -math.inf)
    sink = s["sink"].float().view(h, 1, g, 1) if s["sink"] is not None else z.new_zeros(h, 1, g, 1)
    top = torch.maximum(z.amax(-1, keepdim=True), sink)
    p = torch.exp(z - top)
    p = p / (p.sum(-1, keepdim=True) + torch.exp(sink - top))
    o = torch.matmul(p.view(b, h, t * g, n), v)
    return o.view(b, h, t, g, 64).transpose(1, 2).reshape(b, t, h * g * 64).bfloat16()


def run(s):
    if not own:
        return _plain(s)
    import tritonllm_amd as T

    cache = T.Mxfp4Cache(*s["cache"])
    if s["op"] == "write":
        T.mxfp4_cache_write(cache, s["k"], s["v"], s["offset"], lengths=s["lengths"])
        k, v = T.mxfp4_cache_read(cache, s["first"], s["tokens"])
        return {"k": k, "v": v}
    if s["op"] == "read":
        k, v = T.mxfp4_cache_read(cache, s["first"], s["tokens"])
        return {"k": k, "v": v}
    if s["op"] == "decode":
        return T.mxfp4_attention_decode(s["q"], cache, s["sink"], 0.125, s["window"], s["start"], kv_len_hint=s["keys"])
    return T.mxfp4_attention(s["q"], cache, s["sink"], 0.125, s["window"], s["start"], kv_len_hint=s["keys"])


def work(case):
    if case["op"] in ("write", "read"):
        values = 2 * case["batch"] * case["tokens"] * case["kv_heads"] * case["dim"]
        size = {"bf16": 2, "f16": 2, "f32": 4}[case["type"]] if case["op"] == "write" else 0
        return {"bytes": values * (size + 2) + values * 17 // 32, "flops": 0}
    b, t, n = case["batch"], case["queries"], case["keys"]
    if case["ragged"]:
        n = t + (n - t) // 2                                            # on average
    w = case["window"] or n
    pairs = sum(min(w, n - t + i + 1) for i in range(t))                # keys that the queries of a sequence see
    read = min(n, w + t - 1)
    heads = case["kv_heads"] * case["group"]
    return {"bytes": b * (read * case["kv_heads"] * 2 * 34 + 2 * t * heads * 64 * 2), "flops": 4 * b * pairs * heads * 64}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------
def _values64(blocks, scales):
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
    for i in range(1, 8):
        middle = (FP4[i - 1] + FP4[i]) / 2
        magnitude[(a > middle) | ((a == middle) & (i % 2 == 0))] = FP4[i]
    return (torch.sign(v) * magnitude * 2.0**e).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    kb, ks, vb, vs = s["cache"]
    if case["op"] in ("write", "read"):
        lo, hi = case["first"], case["first"] + case["tokens"]
        k, v = _values64(kb[:, lo:hi], ks[:, lo:hi]), _values64(vb[:, lo:hi], vs[:, lo:hi])
        if case["op"] == "write":
            counts = s["lengths"].tolist() if case["padded"] else [case["tokens"]] * case["batch"]
            for row, count in enumerate(counts):
                k[row, :count] = _quantized64(s["k"][row, :count])
                v[row, :count] = _quantized64(s["v"][row, :count])
        return {"k": k, "v": v}
    # sequence by sequence, the keys that its queries see
    group, heads, t = case["group"], case["kv_heads"] * case["group"], case["queries"]
    starts = s["start"].tolist() * (1 if case["ragged"] else case["batch"])
    out = torch.empty(case["batch"], t, heads, 64, dtype=torch.float64, device="cuda")
    for row, start in enumerate(starts):
        n = start + t
        k = _values64(kb[row, :n], ks[row, :n]).repeat_interleave(group, 1)     # [n, heads, 64]
        v = _values64(vb[row, :n], vs[row, :n]).repeat_interleave(group, 1)
        q = s["q"][row].double().reshape(t, heads, 64)
        for lo in range(0, t, 256):                                             # (for memory)
            z = torch.matmul(q[lo : lo + 256].transpose(0, 1), k.permute(1, 2, 0)) / 8
            far = torch.arange(start + lo, start + lo + z.shape[1], device="cuda")[:, None] - torch.arange(n, device="cuda")
            z[:, (far < 0) | (far >= (case["window"] or n + 1))] = -math.inf
            sink = s["sink"].double() if case["sinks"] else torch.zeros(heads, dtype=torch.float64, device="cuda")
            p = torch.softmax(torch.cat((z, sink[:, None, None].expand(-1, z.shape[1], 1)), 2), 2)[..., :n]
            out[row, lo : lo + 256] = torch.matmul(p, v.transpose(0, 1)).transpose(0, 1)
    return out.reshape(case["batch"], t, heads * 64)
