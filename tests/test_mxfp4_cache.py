"""A KV cache in MXFP4 -- writing, reading back, attention of one and of several new tokens -- against the definitions in float64 on the CPU.

Tolerance of attention. Keys, values and queries are bf16 values, so their products are exact in fp32 and a logit, a sum of 64, is off by at most
64 2^-23 sm_scale sum|q k|; its exponential's argument is rounded twice more, to 2^-23 of its magnitude, and the exponential itself to 2^-22.
A weight is then rounded to bf16 (half a step, 2^-8 of it) ahead of the product with the values, whose fp32 sum over n keys is off by n 2^-23 of
the sum of its magnitudes at most. The denominator sums either the weights or what they were rounded to; in the latter case, with
out = N / Z and roundings d_i, the quotient is off by sum w_i d_i (v_i - out) / Z, at most 2^-8 (A + |out|), A = sum p|v| / Z. The result
is rounded to bf16, 2^-8 of it. So
  |got - want| <= 2^-8 |want| + (1 + 2^-8) ((A + |want|) 2^-8 + A (2 e + n 2^-23)),   e = 64 2^-23 sm_scale max sum|q k| + 2^-22 (max |s| + 16)
(the 2 e for numerator and denominator; 16 covers the running reference, which lies up to 8 powers of two below the largest logit or 7 above it)
and 2^-133 more, twice the rounding of a bf16 value below the smallest normal one, for values of the smallest scales, and n 2^-119 max|v|: a
weight whose fp32 value is below the smallest normal number, 2^-126, may be none at all, and with the reference 7 powers of two above the
largest logit that is one of 2^-119 of its row's largest (of logits hundreds apart: such a weight's value is lost, where the definition still
has e^-83 of it)."""
import ctypes as C
import itertools
import math

import pytest
import torch

import tritonllm_amd as T
from tritonllm_amd import _lib

gpu = pytest.mark.gpu
FP4 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def values(blocks, scales):
    """MXFP4 in float64; a scale byte of 255 is NaN."""
    v = torch.stack((FP4[(blocks & 15).long()], FP4[(blocks >> 4).long()]), -1).flatten(-2)
    p = torch.ldexp(torch.ones((), dtype=torch.float64), scales.long() - 127)
    return (v * torch.where(scales == 255, math.nan, p)[..., None]).flatten(-2)


def quantize_ref(x):
    """codes and scale bytes by search: every level's distance, the even code where two are as near"""
    v = x.double().unflatten(-1, (-1, 32))
    bad = ~v.isfinite().all(-1)
    top = torch.where(bad[..., None], 0.0, v).abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top).exponent.double() - 1, -1000.0).clamp(min=-125) - 2
    a = (torch.where(bad[..., None], 0.0, v) * torch.exp2(-e)[..., None]).abs()
    d = (a[..., None].clamp(max=6) - FP4[:8]).abs() + torch.tensor([0, 1, 0, 1, 0, 1, 0, 1]) * 1e-9      # (odd codes lose ties)
    code = d.argmin(-1) + 8 * torch.signbit(v)
    code[bad] = 0
    code = code.to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.where(bad, 255, (e + 127).long()).to(torch.uint8)


def make_cache(g, batch, slots, heads, dim=64, layout="heads", lo=124, hi=128):
    """A cache of random codes on the GPU: heads outside slots ("heads"), slots outside heads ("slots"), or rows apart from each other
    in a larger buffer ("apart")."""
    out = []
    for _ in range(2):
        for last, top in (((dim // 32, 16), 256), ((dim // 32,), None)):
            rand = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.uint8) if top else torch.randint(lo, hi, s, generator=g, dtype=torch.uint8)
            if layout == "heads":
                t = rand(batch, heads, slots, *last).cuda().transpose(1, 2)
            elif layout == "slots":
                t = rand(batch, slots, heads, *last).cuda()
            else:
                t = rand(batch + 1, heads + 2, slots + 5, *last).cuda()[1:, 1 : heads + 1, 3 : slots + 3].transpose(1, 2)
            out.append(t)
    return T.Mxfp4Cache(*out)


def cpu(cache):
    return [t.cpu().clone() for t in cache]


def attention_ref(q, cache, sinks, scale, window, starts):
    """The definition in float64 and the bound on an answer's error, both [b, t, heads * 64]."""
    kb, ks, vb, vs = cache
    k, v = values(kb, ks), values(vb, vs)
    b, t, h, grp, d = q.shape
    n = k.shape[1]
    want, tol = torch.zeros(b, t, h, grp, d, dtype=torch.float64), torch.zeros(b, t, h, grp, d, dtype=torch.float64)
    sink = torch.zeros(h, grp, dtype=torch.float64) if sinks is None else sinks.double().view(h, grp)
    for row, i in itertools.product(range(b), range(t)):
        p = starts[row] + i
        lo, hi = max(0, p - window + 1) if window else 0, min(p + 1, n)
        if hi <= lo:
            want[row, i] = torch.where((sink == math.inf)[..., None], math.nan, 0.0)
            continue
        qq = q[row, i].double()                                      # [h, grp, d]
        kk, vv = k[row, lo:hi].transpose(0, 1), v[row, lo:hi].transpose(0, 1)      # [h, n, d]
        s = scale * qq @ kk.transpose(1, 2)
        mag = scale * qq.abs() @ kk.abs().transpose(1, 2)
        m = torch.maximum(s.amax(-1), sink)
        w = torch.exp(s - m[..., None])
        z = w.sum(-1) + torch.exp(sink - m)
        want[row, i] = w @ vv / z[..., None]
        a = w @ vv.abs() / z[..., None]
        e = 64 * 2.0**-23 * mag.amax(-1) + 2.0**-22 * (s.abs().amax(-1) + 16)
        tol[row, i] = (2.0**-8 * want[row, i].abs() + (1 + 2.0**-8) * ((a + want[row, i].abs()) * 2.0**-8 + a * (2 * e + (hi - lo) * 2.0**-23)[..., None]) + 2.0**-133
                       + (hi - lo) * 2.0**-119 * vv.abs().nan_to_num().amax())
    return want.view(b, t, -1), tol.view(b, t, -1)


def check(got, want, tol, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in {int(got.isnan().sum())} places, {int(want.isnan().sum())} wanted"
    off = (got - want).abs()
    ok = want.isnan() | (off <= tol)
    assert ok.all(), f"{what}: {int((~ok).sum())} of {ok.numel()} off, by up to {float((off / tol)[~ok].max()):.3g} of the bound"


# ---- writing ----------------------------------------------------------------------------------------------------------------
def write_ref(cache, k, v, offsets, lengths):
    """What a write leaves in a copy of the cache."""
    out = cpu(cache)
    n = out[0].shape[1]
    for x, blocks, scales in ((k, out[0], out[1]), (v, out[2], out[3])):
        codes, sc = quantize_ref(x.cpu())
        for b, t in itertools.product(range(x.shape[0]), range(x.shape[1])):
            if t < lengths[b] and 0 <= offsets[b] + t < n:
                blocks[b, offsets[b] + t], scales[b, offsets[b] + t] = codes[b, t], sc[b, t]
    return out


def same(cache, want):
    return all(torch.equal(a.cpu(), b) for a, b in zip(cache, want))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["heads", "slots", "apart"])
@pytest.mark.parametrize("batch,tokens,slots,heads,dim", [(1, 1, 1, 1, 32), (8, 1, 20, 8, 64), (3, 17, 40, 5, 96), (2, 33, 33, 2, 256), (1, 70, 90, 3, 64)])
def test_write(batch, tokens, slots, heads, dim, layout, dtype):
    g = torch.Generator().manual_seed(batch + tokens + dim)
    cache = make_cache(g, batch, slots, heads, dim, layout, lo=0, hi=256)
    k, v = ((torch.randn(batch, tokens, heads, dim, generator=g) * torch.exp2(torch.randint(-9, 9, (batch, tokens, heads, dim), generator=g).float())).to(dtype)
            for _ in range(2))
    k.view(-1)[3], v.view(-1)[dim - 1] = math.nan, -math.inf
    for offset, lengths in (([slots - tokens], None), ([0], [tokens // 2]), ([int(i) for i in torch.randint(-5, slots + 3, (batch,), generator=g)],
                                                                            [int(i) for i in torch.randint(0, tokens + 1, (batch,), generator=g)])):
        for ints in (torch.int32, torch.int64):
            full = (offset * batch)[:batch]
            want = write_ref(cache, k, v, full, [tokens] * batch if lengths is None else (lengths * batch)[:batch])
            T.mxfp4_cache_write(cache, k.cuda(), v.cuda(), torch.tensor(offset, dtype=ints).cuda(), None if lengths is None else torch.tensor(lengths, dtype=ints).cuda())
            assert same(cache, want), (offset, lengths)


@gpu
def test_write_is_the_quantisation_of_weights():
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(2, 9, 4, 128, generator=g).bfloat16().cuda() for _ in range(2))
    cache = T.mxfp4_cache(2, 9, 4, 128)
    T.mxfp4_cache_write(cache, k, v, torch.zeros(1, dtype=torch.int32, device="cuda"))
    for x, blocks, scales in ((k, cache.k_blocks, cache.k_scales), (v, cache.v_blocks, cache.v_scales)):
        b, s = T.mxfp4_quantize(x)
        assert torch.equal(blocks, b) and torch.equal(scales, s)
    back = T.mxfp4_cache_read(cache)
    assert torch.equal(back[0], T.mxfp4_dequant(cache.k_blocks.contiguous(), cache.k_scales.contiguous()))


@gpu
def test_write_from_strided_and_unaligned_tensors():
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(3, 7, 20, 64, generator=g).bfloat16().cuda()
    odd = torch.empty(3 * 7 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, 7, 4, 64).copy_(wide[:, :, :4])
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    for k, v in ((wide[:, :, 8:12], wide[:, :, 12:16]), (odd, wide[:, :, 4:8]), (wide[:, :, ::5], wide[:, :1, :4].expand(3, 7, 4, 64)),
                 (wide.transpose(2, 3)[:, :, :, :4].transpose(2, 3), wide[..., :4, :].transpose(0, 1).contiguous().transpose(0, 1)),
                 (torch.randn(3, 7, 64, 4, device="cuda").bfloat16().transpose(2, 3), odd)):
        cache = make_cache(g, 3, 9, 4)
        want = write_ref(cache, k, v, [0] * 3, [7] * 3)
        T.mxfp4_cache_write(cache, k, v, zero)
        assert same(cache, want)


@gpu
def test_write_nothing():
    g = torch.Generator().manual_seed(3)
    cache = make_cache(g, 2, 6, 3)
    before = cpu(cache)
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    none = torch.empty(2, 0, 3, 64, dtype=torch.bfloat16, device="cuda")
    T.mxfp4_cache_write(cache, none, none, zero)
    one = torch.ones(2, 4, 3, 64, dtype=torch.bfloat16, device="cuda")
    T.mxfp4_cache_write(cache, one, one, zero, lengths=torch.zeros(2, dtype=torch.int32, device="cuda"))
    T.mxfp4_cache_write(cache, one, one, zero, lengths=torch.tensor([-3], device="cuda"))
    for offset in (6, -4, 2**62, -(2**62), 2**32):
        T.mxfp4_cache_write(cache, one, one, torch.tensor([offset], device="cuda"))
    assert same(cache, before)
    empty = T.mxfp4_cache(2, 0, 3)
    T.mxfp4_cache_write(empty, one, one, zero)
    k, v = T.mxfp4_cache_read(empty)
    assert k.shape == v.shape == (2, 0, 3, 64)


# ---- reading ----------------------------------------------------------------------------------------------------------------
def same_values(got, want):
    """bf16 values that are the wanted ones in float64, NaN and beyond bf16's range included."""
    got, want = got.cpu(), want.to(torch.float32).bfloat16()
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0, posinf=math.inf, neginf=-math.inf), want.nan_to_num(0.0, posinf=math.inf, neginf=-math.inf))


@gpu
@pytest.mark.parametrize("layout", ["heads", "slots", "apart"])
@pytest.mark.parametrize("batch,slots,heads,dim,first,tokens", [(1, 1, 1, 32, 0, 1), (2, 300, 8, 64, 37, 261), (3, 50, 5, 96, 0, None), (2, 70, 3, 160, 69, 1), (1, 2000, 16, 256, 3, 1990),
                                                                (2, 9, 2, 64, 4, 0)])
def test_read(batch, slots, heads, dim, first, tokens, layout):
    g = torch.Generator().manual_seed(slots)
    cache = make_cache(g, batch, slots, heads, dim, layout, lo=0, hi=256)         # every scale byte there is
    kb, ks, vb, vs = cpu(cache)
    k, v = T.mxfp4_cache_read(cache, first, tokens)
    end = slots if tokens is None else first + tokens
    assert k.dtype == torch.bfloat16 and k.shape == (batch, end - first, heads, dim) and k.is_contiguous() and v.is_contiguous()
    assert same_values(k, values(kb, ks)[:, first:end]) and same_values(v, values(vb, vs)[:, first:end])


# ---- attention --------------------------------------------------------------------------------------------------------------
def attention_case(batch, t, heads, group, slots, starts, window=0, sinks=True, layout="heads", seed=0, ints=torch.int64, hint=None, lo=124, hi=128, spread=2.0):
    g = torch.Generator().manual_seed(seed + batch * 7 + t * 5 + heads * 3 + group + slots)
    cache = make_cache(g, batch, slots, heads, layout=layout, lo=lo, hi=hi)
    q = (spread * torch.randn(batch, t, heads, group, 64, generator=g)).bfloat16()
    sink = torch.randn(heads * group, generator=g).bfloat16() if sinks else None
    starts = starts if isinstance(starts, list) else [starts]
    got = T.mxfp4_attention(q.cuda(), cache, None if sink is None else sink.cuda(), 0.125, window, torch.tensor(starts, dtype=ints).cuda(), hint)
    assert got.dtype == torch.bfloat16 and got.is_contiguous()
    want, tol = attention_ref(q, cpu(cache), sink, 0.125, window, (starts * batch)[:batch])
    check(got, want, tol, f"{batch} x {t} queries of {heads} x {group} heads, {slots} slots from {starts}, window {window}")
    if t == 1:
        again = T.mxfp4_attention_decode(q.cuda(), cache, None if sink is None else sink.cuda(), 0.125, window or None, torch.tensor(starts, dtype=ints).cuda(), kv_len_hint=hint)
        assert torch.equal(got, again)


LENGTHS = [0, 1, 14, 15, 16, 30, 31, 32, 33, 62, 63, 64, 100, 127, 128, 129, 255, 256, 300, 511, 700]


@gpu
@pytest.mark.parametrize("group", [1, 5, 8, 9, 16, 17, 40, 64])
def test_one_token_lengths(group):
    for start in LENGTHS:
        attention_case(1, 1, 2, group, 701, start)


@gpu
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 128, 1000])
@pytest.mark.parametrize("group", [8, 12])
def test_one_token_windows(window, group):
    for start in (0, 5, 31, 32, 99, 127, 128, 300, 511):
        attention_case(2, 1, 2, group, 512, start, window=window)


@gpu
@pytest.mark.parametrize("heads,group", [(8, 8), (1, 1), (3, 7), (16, 2), (2, 16), (5, 3)])
@pytest.mark.parametrize("batch", [1, 2, 7, 20])
def test_one_token_of_ragged_rows(batch, heads, group):
    g = torch.Generator().manual_seed(batch + heads)
    starts = [int(i) for i in torch.randint(-2, 400, (batch,), generator=g)]
    starts[0] = 399
    if batch > 2:
        starts[1], starts[2] = -1, 0
    for window, layout, ints in ((0, "heads", torch.int64), (77, "slots", torch.int32), (0, "apart", torch.int64)):
        attention_case(batch, 1, heads, group, 400, starts, window=window, layout=layout, ints=ints, sinks=window == 0)


@gpu
@pytest.mark.parametrize("slots,start", [(5000, 4999), (9001, 8000), (20000, 3), (20000, 150), (4097, 4096), (33000, 32999)])
@pytest.mark.parametrize("hint", [None, 1, 4000, 10**6])
def test_one_token_of_long_caches(slots, start, hint):
    attention_case(1, 1, 2, 8, slots, start, hint=hint)
    attention_case(3, 1, 1, 4, slots, [start, start // 2, 0], hint=hint, window=0)


@gpu
@pytest.mark.parametrize("window", [1025, 1100, 2500, 5000])
@pytest.mark.parametrize("batch,t,heads,group,slots", [(3, 1, 2, 8, 9000), (3, 1, 2, 4, 4000), (3, 1, 2, 12, 9000), (3, 4, 2, 8, 9000), (3, 64, 1, 8, 4001)])
def test_windows_that_workgroups_share(batch, t, heads, group, slots, window):
    """Windows long enough for several workgroups to a stream: rows with all of theirs, with less than is shared out, and with windows that reach past
    either end of the cache."""
    assert shape(batch, t, slots, heads, group, window)[2] > 1
    for layout, starts, sinks in (("heads", [slots - t, 700, 1150], True), ("slots", [slots + window // 3, 3001, window], False), ("apart", [slots + window - 2, 2 * window // 3, -t], True)):
        attention_case(batch, t, heads, group, slots, starts, window=window, layout=layout, sinks=sinks)


@gpu
@pytest.mark.parametrize("t,group,window", [(1, 8, 1100), (1, 8, 0), (1, 12, 2500), (4, 8, 1101), (4, 8, 0), (32, 8, 1100), (32, 8, 0)])
def test_nan_in_walks_that_workgroups_share(t, group, window):
    """Keys and values of NaN just inside and just outside what the first and the last query of a row see, and in the middle."""
    slots, starts = 5000, [4901, 3000, 1177]
    assert shape(3, t, slots, 2, group, window)[2] > 1
    g = torch.Generator().manual_seed(t + window)
    cache = make_cache(g, 3, slots, 2)
    q = torch.randn(3, t, 2, group, 64, generator=g).bfloat16()
    inside = lambda start: start - window + 1 if window else 0
    for row, what, head, half, at in ((0, 3, 0, 1, inside(starts[0])), (0, 3, 1, 0, inside(starts[0]) - 1 if window else starts[0] + t), (0, 1, 1, 0, starts[0] + t - 1), (1, 1, 0, 0, inside(starts[1])),
                                      (1, 3, 1, 1, starts[1]), (1, 3, 1, 0, starts[1] + t), (2, 3, 0, 1, starts[2] - 600), (2, 1, 1, 0, starts[2] + t)):
        cache[what][row, at, head, half] = 255
    want, tol = attention_ref(q, cpu(cache), None, 0.125, window, starts)
    assert want.isnan().any() and not want.isnan().all()
    check(T.mxfp4_attention(q.cuda(), cache, None, 0.125, window, torch.tensor(starts).cuda()), want, tol, f"{t} queries, window {window}")


@gpu
@pytest.mark.parametrize("t", [2, 3, 4, 5, 8, 9, 16, 17, 31, 33, 70])
@pytest.mark.parametrize("heads,group", [(2, 8), (1, 1), (2, 3), (1, 16), (1, 20)])
def test_several_tokens(t, heads, group):
    for start, window in ((0, 0), (3, 0), (130, 0), (130, 40), (29, 1), (200, 128)):
        attention_case(1, t, heads, group, 300, start, window=window)


@gpu
@pytest.mark.parametrize("t", [2, 4, 12, 40, 100, 200])
def test_several_tokens_of_ragged_rows(t):
    for layout, window, ints in (("heads", 0, torch.int32), ("slots", 50, torch.int64), ("apart", 0, torch.int64)):
        attention_case(4, t, 2, 8, 500, [400, 0, -t // 2, 499], window=window, layout=layout, ints=ints)
        attention_case(2, t, 3, 5, 500, [250, 17], window=window, layout=layout, ints=ints, sinks=False)


@gpu
@pytest.mark.parametrize("t,start,slots", [(4, 4092, 4608), (97, 1500, 1600), (64, 3000, 3064), (300, 0, 300), (300, 77, 1000), (257, 1000, 1257), (513, 5, 600)])
@pytest.mark.parametrize("window", [0, 128])
def test_several_tokens_behind_a_past(t, start, slots, window):
    attention_case(1, t, 2, 8, slots, start, window=window)


@gpu
@pytest.mark.parametrize("heads,group", [(1, 8), (2, 1), (1, 3), (2, 5), (1, 12), (1, 16), (1, 33), (1, 64)])
def test_prompts_of_any_group(heads, group):
    for t in (150, 333):
        attention_case(1, t, heads, group, t + 9, 9, window=0)
        attention_case(2, t, heads, group, t, [0, -3], window=60)


def shape(batch, t, slots, heads, group, window=0, hint=0):
    """rows of a run, wavefronts, splits"""
    x = _lib.lib().tllm_mxfp4_attention_shape(batch, t, slots, heads, group, window, hint)
    return x >> 16, x >> 8 & 255, x & 255


def test_shapes():
    """Which kernel serves which sizes, and how many workgroups share the keys."""
    assert shape(1, 1, 300, 8, 8) == (8, 4, 1) and shape(1, 1, 4096, 8, 8, hint=300) == (8, 4, 1)
    assert shape(8, 1, 4096, 8, 8) == (8, 4, 4) and shape(8, 1, 32768, 8, 8) == (8, 4, 8) and shape(49, 1, 2048, 8, 8) == (8, 4, 1)
    assert shape(1, 1, 1 << 29, 1, 1) == (8, 4, 64)
    assert shape(1, 1, 300, 8, 9) == (32, 8, 1) and shape(8, 4, 4096, 8, 8) == (32, 8, 4) and shape(1, 97, 1597, 8, 8) == (32, 8, 1)
    assert shape(1, 256, 2256, 8, 8) == (32, 4, 1) and shape(1, 512, 512, 8, 8) == (64, 4, 1) and shape(1, 512, 8192, 8, 8) == (64, 4, 1)
    assert shape(1, 64, 4096, 8, 8) == (32, 8, 1) and shape(1, 64, 8192, 8, 8) == (32, 8, 2) and shape(2, 72, 11011, 4, 4) == (32, 8, 3)
    assert shape(1, 2048, 2048, 8, 8) == (256, 8, 1) and shape(1, 2048, 8192, 8, 8) == (256, 4, 1) and shape(1, 2048, 8192, 8, 8, hint=2048) == (256, 8, 1) and shape(3, 333, 333, 8, 8) == (128, 4, 1) and shape(1, 1000, 9000, 8, 8) == (128, 4, 1) and shape(1, 2048, 10**6, 8, 8, window=128) == (256, 4, 1)


# (batch, tokens, KV heads, heads of each, slots, run of rows)
KERNELS = [(2, 3, 2, 8, 1500, 32), (24, 6, 8, 8, 90, 32), (30, 7, 8, 8, 70, 32), (50, 16, 8, 8, 60, 64), (24, 40, 8, 8, 120, 256), (16, 150, 16, 1, 200, 128), (64, 3, 4, 60, 50, 128),
           (7, 300, 5, 5, 333, 128), (3, 333, 8, 8, 500, 128), (30, 70, 8, 4, 70, 256), (100, 40, 1, 16, 77, 128)]


@gpu
@pytest.mark.parametrize("batch,t,heads,group,slots,run", KERNELS)
def test_several_tokens_of_each_kernel(batch, t, heads, group, slots, run):
    assert shape(batch, t, slots, heads, group)[0] == run
    g = torch.Generator().manual_seed(batch)
    starts = [int(i) for i in torch.randint(-2, max(slots - t, 1), (batch,), generator=g)]
    attention_case(batch, t, heads, group, slots, starts, sinks=False)
    attention_case(batch, t, heads, group, slots, starts[0] % 20, window=slots // 3, layout="slots", ints=torch.int32)


@gpu
@pytest.mark.parametrize("batch,heads,group,starts,nan", [(1, 16, 5, [0], False), (1, 10, 8, [9], True), (3, 8, 4, [0, -40, 700], True)])
def test_one_long_prompt(batch, heads, group, starts, nan):
    t, slots = 1030, 1100
    assert shape(batch, t, slots, heads, group) == (256, 8, 1)
    g = torch.Generator().manual_seed(heads)
    cache = make_cache(g, batch, slots, heads)
    if nan:                                                    # keys and values of a few places, in either group of wavefronts' shares
        for b, what, at in itertools.product(range(batch), (1, 3), (500, 575, 950)):
            cache[what][b, at + 7 * b, 3, what // 2] = 255
    q = torch.randn(batch, t, heads, group, 64, generator=g).bfloat16()
    want, tol = attention_ref(q, cpu(cache), None, 0.125, 0, starts)
    assert not nan or (want.isnan().any() and not want.isnan().all())
    check(T.mxfp4_attention(q.cuda(), cache, None, 0.125, 0, torch.tensor(starts).cuda()), want, tol, f"prompts at {starts}")


# (batch, tokens, KV heads, heads of each, slots, most keys, {hint: run of rows, wavefronts, splits})
HINTS = [(3, 1, 2, 8, 9000, 4000, {1: (8, 4, 1), 1100: (8, 4, 5), 4000: (8, 4, 16), 10**6: (8, 4, 36)}),
         (8, 4, 2, 8, 4096, 1500, {1: (32, 8, 1), 700: (32, 8, 1), 1500: (32, 8, 6), 10**6: (32, 8, 16)}),
         (3, 32, 2, 8, 5000, 3000, {1: (32, 8, 1), 3000: (32, 8, 5), 10**6: (32, 8, 5)}),
         (24, 40, 8, 8, 1500, 120, {1: (256, 4, 1), 120: (256, 4, 1), 10**6: (64, 4, 1)}),
         (50, 16, 8, 8, 600, 60, {1: (32, 4, 1), 60: (64, 4, 1), 10**6: (64, 4, 1)}),
         (1, 1030, 10, 8, 4096, 1030, {1: (256, 4, 1), 1030: (256, 8, 1), 10**6: (64, 4, 1)})]


@gpu
@pytest.mark.parametrize("batch,t,heads,group,slots,keys,plans", HINTS)
def test_hints_that_change_the_plan(batch, t, heads, group, slots, keys, plans):
    """Hints far below, at and far above the keys that there are: another kernel, another number of splits, an answer within the same bound."""
    g = torch.Generator().manual_seed(slots + t)
    cache = make_cache(g, batch, slots, heads)
    q = (2 * torch.randn(batch, t, heads, group, 64, generator=g)).bfloat16()
    sinks = torch.randn(heads * group, generator=g).bfloat16()
    starts = [keys - t] + [int(i) for i in torch.randint(0, keys - t + 1, (batch - 1,), generator=g)]
    n = max(starts) + t
    want, tol = attention_ref(q, [x[:, :n] for x in cpu(cache)], sinks, 0.125, 0, starts)
    for hint, plan in (*plans.items(), (None, plans[10**6])):
        assert shape(batch, t, slots, heads, group, hint=hint or 0) == plan
        check(T.mxfp4_attention(q.cuda(), cache, sinks.cuda(), 0.125, 0, torch.tensor(starts).cuda(), hint), want, tol, f"hint {hint}, plan {plan}")


@gpu
@pytest.mark.parametrize("t", [1, 3, 20, 200])
def test_attention_past_the_end_and_before_the_beginning(t):
    """Positions beyond the last slot, far beyond it, and before the first."""
    for starts in ([30, -1], [29, -t], [100, -t - 1], [2**31 - 5, -(2**31) + 5], [40, 10]):
        for window in (0, 3, 50, 2**31 - 1):
            attention_case(2, t, 2, 4, 30, starts, window=window, ints=torch.int32)
    attention_case(2, t, 2, 4, 30, [2**62, -(2**62)], window=7)
    attention_case(2, t, 2, 4, 30, [2**40, -(2**40)])


@gpu
@pytest.mark.parametrize("t", [1, 4, 200])
def test_attention_of_smallest_and_largest_scales(t):
    """Keys so small that every logit is 0, values near both ends of bf16's range, logits that reach hundreds."""
    attention_case(2, t, 2, 8, 300, 250 if t < 50 else 40, lo=0, hi=6)
    attention_case(2, t, 2, 8, 300, 250 if t < 50 else 40, lo=130, hi=134)
    g = torch.Generator().manual_seed(t)
    for lo, hi in ((0, 4), (235, 240)):
        kb, ks, _, _ = make_cache(g, 1, 300, 2)
        _, _, vb, vs = make_cache(g, 1, 300, 2, lo=lo, hi=hi)
        cache = T.Mxfp4Cache(kb, ks, vb, vs)
        q = torch.randn(1, t, 2, 8, 64, generator=g).bfloat16()
        want, tol = attention_ref(q, cpu(cache), None, 0.125, 0, [60])
        check(T.mxfp4_attention(q.cuda(), cache, None, 0.125, 0, torch.tensor([60]).cuda()), want, tol, f"values of scale bytes {lo} to {hi}")


@gpu
@pytest.mark.parametrize("t,group,heads,pairs", [(1, 8, 2, 1), (1, 16, 2, 1), (4, 8, 2, 1), (33, 4, 2, 1), (200, 8, 2, 1), (100, 4, 8, 8), (100, 4, 8, 32)])
def test_what_is_not_seen_does_not_matter(t, group, heads, pairs):
    """Slots of NaN, of the largest values and of infinite ones outside what the queries see."""
    g = torch.Generator().manual_seed(t)
    for start, window in ((0, 0), (40, 0), (40, 16), (45, 7)):
        cache = make_cache(g, 2 * pairs, 300, heads)
        q = torch.randn(2 * pairs, t, heads, group, 64, generator=g).bfloat16().cuda()
        at = torch.tensor([start, start + 3] * pairs).cuda()
        first = T.mxfp4_attention(q, cache, None, 0.125, window, at)
        assert first.isfinite().all()
        for byte in (255, 254, 252):
            for b, s in enumerate((start, start + 3) * pairs):
                cache.k_scales[b, s + t :] = byte
                cache.v_scales[b, s + t :] = byte
                if window:
                    cache.k_scales[b, : max(0, s - window + 1)] = byte
                    cache.v_scales[b, : max(0, s - window + 1)] = byte
            assert torch.equal(T.mxfp4_attention(q, cache, None, 0.125, window, at), first)


@gpu
@pytest.mark.parametrize("t,group", [(1, 8), (1, 16), (4, 8), (33, 4), (100, 1), (200, 8), (400, 8)])
def test_nan_reaches_who_sees_it(t, group):
    """A block of 32 keys or of 32 values of NaN: who sees a key of it gets nothing but NaN, who sees a value of it gets NaN in its half of the
    head, and no other query does."""
    for window in (0, 20):
        for where in (0, 30, 64, 70, 95):
            for half, what in itertools.product((0, 1), (1, 3)):
                g = torch.Generator().manual_seed(where)
                cache = make_cache(g, 1, 500, 2)
                cache[what][0, where, 1, half] = 255
                q = torch.randn(1, t, 2, group, 64, generator=g).bfloat16()
                want, tol = attention_ref(q, cpu(cache), None, 0.125, window, [64])
                check(T.mxfp4_attention(q.cuda(), cache, None, 0.125, window, torch.tensor([64]).cuda()), want, tol, f"{t} queries, window {window}, NaN at {where}")


@gpu
@pytest.mark.parametrize("batch,t,group,run", [(24, 40, 8, 256), (10, 70, 8, 128), (50, 16, 8, 64), (30, 7, 8, 32)])
def test_nan_in_a_batch_of_each_kernel(batch, t, group, run):
    assert shape(batch, t, 150, 8, group)[0] == run
    for window in (0, 25):
        g = torch.Generator().manual_seed(run)
        cache = make_cache(g, batch, 150, 8)
        for b in range(batch):                                 # somewhere in each row: a block of keys, of values, of both, of neither
            for what in (1, 3):
                if int(torch.randint(0, 3, (), generator=g)):
                    cache[what][b, int(torch.randint(0, 110, (), generator=g)), int(torch.randint(0, 8, (), generator=g)), int(torch.randint(0, 2, (), generator=g))] = 255
        q = torch.randn(batch, t, 8, group, 64, generator=g).bfloat16()
        starts = [int(i) for i in torch.randint(0, 110 - t, (batch,), generator=g)]
        want, tol = attention_ref(q, cpu(cache), None, 0.125, window, starts)
        assert want.isnan().any() and not want.isnan().all()
        check(T.mxfp4_attention(q.cuda(), cache, None, 0.125, window, torch.tensor(starts).cuda()), want, tol, f"runs of {run}, window {window}")


@gpu
@pytest.mark.parametrize("batch,t,heads,group,slots,run", [(1, 4, 2, 8, 100, (32, 8)), (2, 33, 2, 4, 120, (32, 8)), (30, 7, 8, 8, 70, (32, 4)), (50, 16, 8, 8, 60, (64, 4)), (100, 40, 1, 16, 77, (128, 4)),
                                                           (24, 40, 8, 8, 120, (256, 4)), (1, 1030, 10, 8, 1100, (256, 8))])
def test_infinite_values_reach_who_sees_them(batch, t, heads, group, slots, run):
    """One slot of each row whose 32 values of one half of one head read as infinite in every other place (2^128 and more of scale bytes 253 and
    254), and as large finite ones or as zeros between. Queries ahead of the slot, or past it with a window, have the answer without it; those
    that see it have nothing finite in the infinite places, with the sign of the infinity unless it is NaN, and the definition's answer in all others."""
    assert shape(batch, t, slots, heads, group)[:2] == run
    g = torch.Generator().manual_seed(batch + t)
    plain = make_cache(g, batch, slots, heads)
    q = torch.randn(batch, t, heads, group, 64, generator=g).bfloat16()
    start = 9
    cases = [(0, start + t // 2, 253, 3), (0, start + t - 1, 254, 1), (12, start + t // 2, 253, 0), (12, start - 5, 254, 0), (0, start - 5, 253, 1)]
    for window, slot, byte, finite in cases if t < 1000 else cases[::2]:
        half, head = slot % 2, t % heads
        codes = torch.tensor([7, finite, 14, finite + 8] * 8, dtype=torch.uint8)      # 6 and -4: infinite; between them the code `finite`, of either sign
        infinite = torch.tensor([True, False] * 16)
        cache, without, between = ([x.clone() for x in plain] for _ in range(3))
        for c, kept, power in ((cache, codes, byte), (without, 0 * codes, 0), (between, torch.where(infinite, 0, codes), byte)):
            c[0][:, slot, head] = 0                                 # a key of zeros: its weight is about 1 at most, and the finite values' sums stay finite
            c[2][:, slot, head, half] = (kept[0::2] | kept[1::2] << 4).cuda()
            c[3][:, slot, head, half] = power
        got = T.mxfp4_attention(q.cuda(), T.Mxfp4Cache(*cache), None, 0.125, window, torch.tensor([start]).cuda())
        want, tol = (x.view(batch, t, heads, group, 64) for x in attention_ref(q, cpu(without), None, 0.125, window, [start] * batch))
        with_between = [x.view(batch, t, heads, group, 64) for x in attention_ref(q, cpu(between), None, 0.125, window, [start] * batch)]
        at = start + torch.arange(t)
        sees = (slot <= at) & (slot > at - window if window else slot >= 0)
        assert sees.any() and (window or slot < start or not sees.all())
        got = got.cpu().double().view(batch, t, heads, group, 64).clone()
        piece = got[:, sees, head, :, 32 * half : 32 * half + 32]
        assert not piece[..., infinite].isfinite().any()
        sign = torch.tensor([1.0, -1.0] * 8, dtype=torch.float64)   # (of the infinite places)
        assert (piece[..., infinite].isnan() | (piece[..., infinite] == sign * math.inf)).all()
        for x, y in zip((want, tol), with_between):                 # the finite values of the piece: the bound of their own sums, for their own columns alone
            x[:, sees, head, :, 32 * half : 32 * half + 32] = y[:, sees, head, :, 32 * half : 32 * half + 32]
        columns = torch.arange(32 * half, 32 * half + 32)[infinite]
        for x in (got, want, tol):
            x[:, sees.nonzero()[:, None], head, :, columns[None, :]] = 0
        check(got.reshape(batch, t, -1), want.reshape(batch, t, -1), tol.reshape(batch, t, -1), f"byte {byte} at {slot}, window {window}, {finite} between")


@gpu
@pytest.mark.parametrize("batch,t,heads,group,slots,window", [(2, 1, 2, 8, 90, 0), (2, 1, 2, 16, 90, 30), (2, 5, 2, 8, 100, 0), (1, 33, 1, 12, 120, 20), (30, 7, 8, 8, 70, 0), (50, 16, 8, 8, 60, 12), (100, 40, 1, 16, 77, 0),
                                                              (24, 40, 8, 8, 120, 0), (24, 40, 8, 8, 120, 25), (1, 70, 2, 8, 3000, 0)])
def test_nan_and_infinities_together(batch, t, heads, group, slots, window):
    """Several pieces of NaN and of infinities in each row, some of them neighbours: a query has NaN where it sees NaN, nothing finite where it sees an
    infinity, and the definition's answer everywhere else."""
    g = torch.Generator().manual_seed(slots + t + window)
    pick = lambda n: int(torch.randint(0, n, (), generator=g))
    start = slots - t if slots > 1000 else 9
    plain = make_cache(g, batch, slots, heads)
    q = torch.randn(batch, t, heads, group, 64, generator=g).bfloat16()
    at = start + torch.arange(t)
    cache, without = [x.cpu().clone() for x in plain], [x.cpu().clone() for x in plain]
    for b in range(batch):
        first = max(0, start + t - 40) if slots > 1000 else 0
        places = {(first + pick(start + t + 3 - first), pick(heads), pick(2)) for _ in range(3)}
        n, h, half = next(iter(places))
        places |= {(n + 1, h, half), (n, h, 1 - half)}              # (its neighbours)
        for n, h, half in sorted(places):
            n = min(n, slots - 1)
            byte = (253, 254, 255)[pick(3)]
            which = torch.rand(32, generator=g) < 0.3
            codes = torch.where(which, torch.tensor((7, 14, 15, 6))[torch.randint(0, 4, (32,), generator=g)], 0).to(torch.uint8)
            cache[2][b, n, h, half], cache[3][b, n, h, half] = codes[0::2] | codes[1::2] << 4, byte
            without[2][b, n, h, half], without[3][b, n, h, half] = 0, 0
    v = values(cache[2], cache[3])                                  # [batch, slots, heads, 64]
    key = torch.arange(slots)
    sees = (key <= at[:, None]) & (key > at[:, None] - window if window else key >= 0)
    nan = torch.einsum("tn,bnhd->bthd", sees.float(), v.isnan().float()) > 0
    infinite = torch.einsum("tn,bnhd->bthd", sees.float(), (v.abs() >= 2.0**128).float()) > 0
    got = T.mxfp4_attention(q.cuda(), T.Mxfp4Cache(*(x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in cache)), None, 0.125, window, torch.tensor([start]).cuda())
    want, tol = attention_ref(q, without, None, 0.125, window, [start] * batch)
    wide = lambda x: x[:, :, :, None].expand(batch, t, heads, group, 64).reshape(batch, t, -1)
    got = got.cpu().double()
    assert got[wide(nan)].isnan().all() and not got[wide(infinite)].isfinite().any()
    for x in (got, want, tol):
        x[wide(nan | infinite)] = 0
    check(got, want, tol, f"{t} queries, window {window}")


@gpu
@pytest.mark.parametrize("batch,t,heads,group,slots", [(1, 4, 2, 8, 100), (50, 16, 8, 8, 60), (100, 40, 1, 16, 77), (24, 40, 8, 8, 120)])
def test_infinite_keys_are_nothing_to_who_does_not_see_them(batch, t, heads, group, slots):
    g = torch.Generator().manual_seed(batch + t)
    plain = make_cache(g, batch, slots, heads)
    q = torch.randn(batch, t, heads, group, 64, generator=g).bfloat16()
    for window, slot, byte in ((0, 9 + t // 2, 254), (12, 9 + t // 2, 253), (12, 7, 254)):
        cache = [x.clone() for x in plain]
        cache[1][:, slot] = byte
        got = T.mxfp4_attention(q.cuda(), T.Mxfp4Cache(*cache), None, 0.125, window, torch.tensor([9]).cuda())
        want, tol = attention_ref(q, cpu(plain), None, 0.125, window, [9] * batch)
        at = 9 + torch.arange(t)
        other = (slot > at) | (slot <= at - window if window else slot < 0)
        if other.any():
            check(got[:, other], want[:, other], tol[:, other], f"byte {byte} at {slot}, window {window}")


@gpu
def test_nan_and_infinite_queries_stay_with_their_row():
    g = torch.Generator().manual_seed(4)
    for t, group in ((1, 8), (5, 4), (200, 4)):
        cache = make_cache(g, 2, 300, 2)
        q = torch.randn(2, t, 2, group, 64, generator=g).bfloat16()
        at = torch.tensor([60, 33]).cuda()
        first = T.mxfp4_attention(q.cuda(), cache, None, 0.125, 0, at)
        q[0, t - 1, 1, group - 1, 5] = math.nan
        q[1, 0, 0, 1] = math.inf
        got = T.mxfp4_attention(q.cuda(), cache, None, 0.125, 0, at).view(2, t, 2, group, 64)
        for b, i, h, j in ((0, t - 1, 1, group - 1), (1, 0, 0, 1)):
            assert got[b, i, h, j].isnan().all()
            got[b, i, h, j] = first.view_as(got)[b, i, h, j]
        assert torch.equal(got.view_as(first), first)


@gpu
@pytest.mark.parametrize("t", [1, 4, 200])
def test_sinks(t):
    """Sinks that leave the keys nothing, sinks that count for nothing, and no key at all beside either."""
    g = torch.Generator().manual_seed(5)
    cache = make_cache(g, 2, 200, 1)
    q = torch.randn(2, t, 1, 4, 64, generator=g).bfloat16()
    sink = torch.tensor([-math.inf, 1000.0, -1000.0, torch.finfo(torch.bfloat16).min]).bfloat16()
    for starts in ([100, 3], [-t, 0], [-t - 5, -t]):
        got = T.mxfp4_attention(q.cuda(), cache, sink.cuda(), 0.125, 0, torch.tensor(starts).cuda())
        plain, tol = attention_ref(q, cpu(cache), sink, 0.125, 0, starts)
        check(got, plain, tol, f"sinks from {starts}")
        for b in range(2):
            if starts[b] + t <= 0:
                assert got[b].eq(0).all()


@gpu
def test_a_cache_that_rows_share():
    """A prefix that all rows see, as one copy of it."""
    g = torch.Generator().manual_seed(6)
    one = make_cache(g, 1, 300, 2)
    cache = T.Mxfp4Cache(*(t.expand(5, *t.shape[1:]) for t in one))
    for t in (1, 3, 150):
        q = torch.randn(5, t, 2, 8, 64, generator=g).bfloat16()
        starts = [299 - t, 0, 17, 200, 100]
        want, tol = attention_ref(q, cpu(cache), None, 0.125, 0, starts)
        check(T.mxfp4_attention(q.cuda(), cache, None, 0.125, 0, torch.tensor(starts).cuda()), want, tol)
    k, _ = T.mxfp4_cache_read(cache, 3, 9)
    assert same_values(k, values(*cpu(cache)[:2])[:, 3:12])
    x = torch.ones(5, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="share memory"):
        T.mxfp4_cache_write(cache, x, x, torch.zeros(1, dtype=torch.int64, device="cuda"))


@gpu
@pytest.mark.parametrize("t", [1, 5, 150])
def test_queries_from_strides(t):
    g = torch.Generator().manual_seed(7)
    cache = make_cache(g, 3, 200, 4)
    wide = torch.randn(3, t, 4 * 8 * 64 + 2 * 4 * 64, generator=g).bfloat16()            # as the QKV projection writes it
    q = wide[..., : 4 * 8 * 64].view(3, t, 4, 8, 64)
    want, tol = attention_ref(q, cpu(cache), None, 0.3, 0, [49] * 3)
    at = torch.tensor([49]).cuda()
    dev = wide.cuda()[..., : 4 * 8 * 64].view(3, t, 4, 8, 64)
    odd = torch.empty(dev.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(dev.shape).copy_(dev)
    for x in (dev, odd, dev.transpose(2, 3).contiguous().transpose(2, 3), dev.transpose(0, 1).contiguous().transpose(0, 1)):
        check(T.mxfp4_attention(x, cache, None, 0.3, 0, at), want, tol)


@gpu
@pytest.mark.parametrize("t", [1, 4, 200])
def test_scales_at_odd_addresses(t):
    g = torch.Generator().manual_seed(13)
    cache = make_cache(g, 2, 90, 2)

    def odd(s):
        s = s.transpose(1, 2)
        return torch.empty(s.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(s.shape).copy_(s).transpose(1, 2)

    cache = cache._replace(k_scales=odd(cache.k_scales), v_scales=odd(cache.v_scales))
    k, v = torch.randn(2, 2, 2, 64, generator=g).bfloat16().cuda(), torch.randn(2, 2, 2, 64, generator=g).bfloat16().cuda()
    T.mxfp4_cache_write(cache, k, v, torch.tensor([11, 40]).cuda())
    assert same_values(T.mxfp4_cache_read(cache)[0], values(*cpu(cache)[:2]))
    q = torch.randn(2, t, 2, 8, 64, generator=g).bfloat16()
    want, tol = attention_ref(q, cpu(cache), None, 0.125, 0, [89, 44])
    check(T.mxfp4_attention(q.cuda(), cache, None, 0.125, 0, torch.tensor([89, 44]).cuda(), 2**70), want, tol)


@gpu
def test_slots_beyond_32_bits():
    """Slots 16 MB apart: 300 of them span 5 GB, and the offsets of a cache's end pass 32 bits."""
    n, far = 300, 2**24 - 16
    g = torch.Generator().manual_seed(8)
    buffer = torch.zeros(n * far + 4096, dtype=torch.uint8, device="cuda")
    view = lambda at, *last: buffer[at:].as_strided((1, n, 1, *last), (0, far, 0, *((16, 1) if len(last) == 2 else (1,))))
    cache = T.Mxfp4Cache(view(0, 2, 16), view(64, 2), view(32, 2, 16), view(72, 2))
    k, v = (torch.randn(1, n, 1, 64, generator=g).bfloat16() for _ in range(2))
    T.mxfp4_cache_write(cache, k.cuda(), v.cuda(), torch.zeros(1, dtype=torch.int64, device="cuda"))
    (kb, ks), (vb, vs) = quantize_ref(k), quantize_ref(v)
    got = T.mxfp4_cache_read(cache)
    assert same_values(got[0], values(kb, ks)) and same_values(got[1], values(vb, vs))
    for t in (1, 4, 200):
        q = torch.randn(1, t, 1, 8, 64, generator=g).bfloat16()
        want, tol = attention_ref(q, [kb, ks, vb, vs], None, 0.125, 0, [n - t])
        check(T.mxfp4_attention(q.cuda(), cache, None, 0.125, 0, torch.tensor([n - t]).cuda()), want, tol)
    q = torch.randn(1, 64, 1, 8, 64, generator=g).bfloat16()
    want, tol = attention_ref(q, [kb, ks, vb, vs], None, 0.125, 0, [n - 64])
    for batch, run in ((100, 128), (140, 256)):                     # the same for many rows, all over the one cache
        assert shape(batch, 64, n, 1, 8)[0] == run
        got = T.mxfp4_attention(q.cuda().expand(batch, 64, 1, 8, 64), T.Mxfp4Cache(*(x.expand(batch, *x.shape[1:]) for x in cache)), None, 0.125, 0, torch.tensor([n - 64]).cuda())
        check(got[:1], want, tol)
        assert torch.equal(got, got[:1].expand_as(got))
    del buffer
    torch.cuda.empty_cache()


@gpu
def test_nothing_to_attend_with():
    cache = T.mxfp4_cache(0, 9, 2)
    at = torch.zeros(1, dtype=torch.int64, device="cuda")
    assert T.mxfp4_attention(torch.empty(0, 1, 2, 8, 64, dtype=torch.bfloat16, device="cuda"), cache, None, 0.125, 0, at).shape == (0, 1, 1024)
    cache = T.mxfp4_cache(2, 9, 2)
    assert T.mxfp4_attention(torch.empty(2, 0, 2, 8, 64, dtype=torch.bfloat16, device="cuda"), cache, None, 0.125, 0, at).shape == (2, 0, 1024)


# ---- together, in graphs, on streams ------------------------------------------------------------------------------------------
def step(x, w, bias, yarn, cache, sinks, positions, offset, start):
    """A decode step's attention half: projection and rotary, the new token into the cache, attention over it."""
    b = x.shape[0]
    q, k, v = T.qkv_rope_forward(x, w, bias, 16, 2, 64, yarn=yarn, positions=positions)
    T.mxfp4_cache_write(cache, k.view(b, 1, 2, 64), v.view(b, 1, 2, 64), offset)
    return T.mxfp4_attention_decode(q.view(b, 1, 2, 8, 64), cache, sinks, 0.125, None, start)


def step_inputs(g, batch):
    w = (0.05 * torch.randn(20 * 64, 256, generator=g)).bfloat16().cuda()
    return w, torch.randn(20 * 64, generator=g).bfloat16().cuda(), T.gpt_oss_yarn(), torch.randn(16, generator=g).bfloat16().cuda()


@gpu
def test_a_prompt_and_tokens_behind_it():
    """A padded batch of two prompts, then tokens, all through the cache: attention as over what the cache reads back as."""
    g = torch.Generator().manual_seed(9)
    w, bias, yarn, sinks = step_inputs(g, 2)
    cache = T.mxfp4_cache(2, 64, 2)
    lengths = torch.tensor([20, 13]).cuda()
    x = torch.randn(2 * 20, 256, generator=g).bfloat16().cuda()
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    q, k, v = T.qkv_rope_forward(x, w, bias, 16, 2, 64, yarn=yarn, tokens_per_batch=20)
    T.mxfp4_cache_write(cache, k.view(2, 20, 2, 64), v.view(2, 20, 2, 64), zero, lengths)
    o = T.mxfp4_attention(q.view(2, 20, 2, 8, 64), cache, sinks, 0.125, 0, zero)
    want, tol = attention_ref(q.view(2, 20, 2, 8, 64).cpu(), cpu(cache), sinks.cpu(), 0.125, 0, [0, 0])
    check(o, want, tol)
    kc, vc = T.mxfp4_cache_read(cache)
    other = T.attention(q.view(2, 20, 2, 8, 64).contiguous(), kc, vc, sinks, 0.125, 0, zero)      # the same over bf16 keys and values
    assert (other.double().cpu() - want).abs().le(tol + 2.0**-8 * want.abs()).all()
    assert cache.k_blocks[1, 13:].eq(0).all() and cache.k_blocks[0, 19].ne(0).any()
    at = lengths.clone()
    for i in range(3):
        tok = torch.randn(2, 256, generator=g).bfloat16().cuda()
        o = step(tok, w, bias, yarn, cache, sinks, at, at, at)
        q, _, _ = T.qkv_rope_forward(tok, w, bias, 16, 2, 64, yarn=yarn, positions=at)
        want, tol = attention_ref(q.view(2, 1, 2, 8, 64).cpu(), cpu(cache), sinks.cpu(), 0.125, 0, at.tolist())
        check(o, want, tol)
        at += 1


@gpu
def test_steps_in_a_graph():
    """A captured step follows positions on the device, replay after replay, with eager work between."""
    g = torch.Generator().manual_seed(10)
    w, bias, yarn, sinks = step_inputs(g, 3)
    make = lambda: T.mxfp4_cache(3, 2000, 2)
    a, b = make(), make()
    x, at = torch.randn(3, 256, generator=g).bfloat16().cuda(), torch.tensor([5, 0, 1500]).cuda()
    step(x, w, bias, yarn, make(), sinks, at, at, at)                 # (loads the kernels)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, w, bias, yarn, a, sinks, at, at, at)
        drafts = T.mxfp4_attention(got.view(3, 1, 2, 8, 64).expand(3, 4, 2, 8, 64), a, sinks, 0.125, 300, at)
    for i in range(5):
        x.copy_(torch.randn(3, 256, generator=g).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        want = step(x, w, bias, yarn, b, sinks, at, at, at)
        assert torch.equal(got, want), i
        assert torch.equal(drafts, T.mxfp4_attention(want.view(3, 1, 2, 8, 64).expand(3, 4, 2, 8, 64), b, sinks, 0.125, 300, at))
        assert all(torch.equal(p, r) for p, r in zip(a, b))
        at += 7


@gpu
def test_two_graphs_and_two_streams():
    """Calls that overlap keep to their own workspaces and outputs."""
    g = torch.Generator().manual_seed(11)
    caches = [make_cache(g, 2, 3000, 2) for _ in range(2)]
    qs = [torch.randn(2, 1, 2, 8, 64, generator=g).bfloat16().cuda() for _ in range(2)]
    at = torch.tensor([2999, 1700]).cuda()
    want = [T.mxfp4_attention(q, c, None, 0.125, 0, at) for q, c in zip(qs, caches)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(T.mxfp4_attention(qs[i], caches[i], None, 0.125, 0, at))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])
    graphs, got = [], []
    for q, c in zip(qs, caches):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(T.mxfp4_attention(q, c, None, 0.125, 0, at))
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_the_same_each_time():
    g = torch.Generator().manual_seed(12)
    cache = make_cache(g, 4, 4000, 8)
    for t in (1, 3, 97, 300):
        q = torch.randn(4, t, 8, 8, 64, generator=g).bfloat16().cuda()
        at = torch.tensor([3700, 5, 900, 2222]).cuda()
        first = T.mxfp4_attention(q, cache, None, 0.125, 0, at)
        assert all(torch.equal(T.mxfp4_attention(q, cache, None, 0.125, 0, at), first) for _ in range(5))


# ---- refusals -----------------------------------------------------------------------------------------------------------------
def descriptor(**other):
    fields = dict(k_blocks=4096, k_scales=8192, v_blocks=12288, v_scales=16384, batch_stride=3200, slot_stride=32, head_stride=1600, scale_batch_stride=200,
                  scale_slot_stride=2, scale_head_stride=100, batch=2, n_slots=50, n_kv_heads=2, head_dim=64)
    return _lib.TllmMxCache(**{**fields, **other})


def test_struct_layout_matches_header():
    assert C.sizeof(_lib.TllmMxCache) == 4 * 8 + 8 * 8 + 2 * 4


def test_entry_points_refuse_what_they_cannot_do():
    lib = _lib.lib()
    said = lambda: lib.tllm_last_error().decode()
    ints = lambda *v: (C.c_int64 * 3)(*v)
    p = 1 << 20                                                     # (an address that no call here comes to use)

    def write(cache=None, k=p, v=p, kind=0, ks=(128, 128, 64), vs=(128, 128, 64), tokens=1, offset=p):
        return lib.tllm_mxfp4_cache_write(C.byref(cache or descriptor()), k, v, kind, ints(*ks), ints(*vs), tokens, offset, 1, 0, None, 0, 0, None)

    def read(cache=None, first=0, tokens=1, k=p, v=p):
        return lib.tllm_mxfp4_cache_read_bf16(C.byref(cache or descriptor()), first, tokens, k, v, None)

    def attend(cache=None, q=p, qbs=1024, qts=1024, sinks=None, out=p, obs=1024, ots=1024, n_q=1, group=8, scale=0.125, window=0, start=p, hint=0, work=None, size=0):
        return lib.tllm_mxfp4_attention_bf16(q, qbs, qts, C.byref(cache or descriptor()), sinks, out, obs, ots, n_q, group, scale, window, start, 1, 0, hint, work, size, None)

    assert lib.tllm_mxfp4_cache_write(None, p, p, 0, ints(1, 1, 1), ints(1, 1, 1), 1, p, 1, 0, None, 0, 0, None) == -1 and "NULL" in said()
    for call in (write, read, attend):
        for bad, code in ((dict(batch=-1), -2), (dict(batch=70000), -2), (dict(n_slots=2**30), -2), (dict(n_kv_heads=0), -2), (dict(head_dim=48), -2), (dict(head_dim=0), -2),
                          (dict(head_dim=2048), -2), (dict(k_blocks=None), -1), (dict(v_scales=None), -1), (dict(v_blocks=4100), -3), (dict(slot_stride=40), -3),
                          (dict(head_stride=-16), -2), (dict(slot_stride=2**24), -2), (dict(scale_slot_stride=2**24), -2)):
            assert call(cache=descriptor(**bad)) == code and said(), (call, bad)
    for bad, code in ((dict(k=None), -1), (dict(v=None), -1), (dict(offset=None), -1), (dict(kind=3), -1), (dict(tokens=-1), -1), (dict(k=p + 8), -3), (dict(vs=(128, 130, 64)), -3),
                      (dict(cache=descriptor(batch_stride=0)), -1), (dict(cache=descriptor(scale_head_stride=0)), -1), (dict(cache=descriptor(slot_stride=0)), -1)):
        assert write(**bad) == code and said(), bad
    assert write(tokens=0) == 0 and write(cache=descriptor(batch=0)) == 0 and write(cache=descriptor(n_slots=0)) == 0
    for bad, code in ((dict(first=-1), -2), (dict(tokens=-1), -2), (dict(first=50), -2), (dict(first=20, tokens=31), -2), (dict(first=2**62, tokens=2**62), -2), (dict(k=None), -1),
                      (dict(v=p + 2), -3)):
        assert read(**bad) == code and said(), bad
    assert read(first=50, tokens=0) == 0 and read(cache=descriptor(batch=0)) == 0
    for bad, code in ((dict(cache=descriptor(head_dim=128)), -2), (dict(cache=descriptor(n_slots=0)), -2), (dict(n_q=-1), -2), (dict(n_q=2**24), -2), (dict(group=0), -2), (dict(group=65), -2),
                      (dict(window=-1), -1), (dict(scale=0.0), -1), (dict(scale=-1.0), -1), (dict(scale=math.nan), -1), (dict(scale=math.inf), -1), (dict(hint=-1), -1), (dict(q=None), -1),
                      (dict(out=None), -1), (dict(start=None), -1), (dict(q=p + 2), -3), (dict(qts=1028), -3), (dict(out=p + 8), -3),
                      (dict(cache=descriptor(n_slots=100000)), -1)):                      # (splits: a workspace is needed)
        assert attend(**bad) == code and said(), bad
    assert attend(n_q=0) == 0 and attend(cache=descriptor(batch=0)) == 0
    need = lib.tllm_mxfp4_attention_workspace_bytes(2, 1, 100000, 2, 8, 0, 0)
    assert need > 0 and attend(cache=descriptor(n_slots=100000), work=p, size=need - 1) == -1 and "workspace" in said()
    assert lib.tllm_mxfp4_attention_workspace_bytes(2, 1, 100000, 2, 8, 0, 100) < need and lib.tllm_mxfp4_attention_shape(0, 1, 10, 1, 1, 0, 0) == 0
    assert lib.tllm_mxfp4_attention_shape(1, 1, 2**30, 1, 1, 0, 0) == 0 and lib.tllm_mxfp4_attention_workspace_bytes(1, 2**24, 10, 1, 1, 0, 0) == 0


def test_ops_refuse_cpu_tensors():
    cache = T.mxfp4_cache(1, 4, 2, device="cpu")
    x, at = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int64)
    for call in (lambda: T.mxfp4_cache_write(cache, x, x, at), lambda: T.mxfp4_cache_read(cache), lambda: T.mxfp4_attention(x[:, :, :, None], cache, None, 1.0, 0, at),
                 lambda: T.mxfp4_attention_decode(x[:, :, :, None], cache, None, 1.0, 0, at)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(AssertionError):
        T.mxfp4_cache(1, 4, 2, head_dim=40, device="cpu")


@gpu
def test_ops_refuse_wrong_types_and_shapes():
    cache = T.mxfp4_cache(2, 10, 3)
    x, at = torch.zeros(2, 1, 3, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    q = torch.zeros(2, 1, 3, 4, 64, dtype=torch.bfloat16, device="cuda")
    kb, ks, vb, vs = cache
    bad_caches = [(kb, ks, vb[:, :9], vs[:, :9]), (kb, ks[:, :9], vb, vs), (kb.short(), ks, vb, vs), (kb, ks.float(), vb, vs), (kb, ks, vb.contiguous(), vs), (kb[..., :8], ks, vb[..., :8], vs),
                  (kb.flip(4).transpose(3, 4), ks, vb, vs), (kb, ks, vb, vs.contiguous()), (kb[:, :, :, :0], ks[:, :, :, :0], vb[:, :, :, :0], vs[:, :, :, :0])]
    for bad in bad_caches:
        for call in (lambda: T.mxfp4_cache_write(bad, x, x, at), lambda: T.mxfp4_cache_read(bad), lambda: T.mxfp4_attention(q, bad, None, 1.0, 0, at)):
            with pytest.raises(AssertionError):
                call()
    for k, v, offset, lengths in ((x.double(), x.double(), at, None), (x, x.float(), at, None), (x, x[:, :0], at, None), (x[:1], x[:1], at, None), (x[..., :32], x[..., :32], at, None),
                                  (x[:, :, :2], x[:, :, :2], at, None), (x[0], x[0], at, None), (x, x, at.float(), None), (x, x, at[0], None), (x, x, at.expand(3), None),
                                  (x, x, at[:0], None), (x, x, at, at.expand(3)), (x, x, at, at.short())):
        with pytest.raises(AssertionError):
            T.mxfp4_cache_write(cache, k, v, offset, lengths)
    for first, tokens in ((-1, 3), (11, None), (0, 11), (4, -1), (4, 7)):
        with pytest.raises(AssertionError):
            T.mxfp4_cache_read(cache, first, tokens)
    sinks = torch.zeros(12, dtype=torch.bfloat16, device="cuda")
    for qq, s, start in ((q.float(), sinks, at), (q[0], sinks, at), (q[:1], sinks, at), (q[:, :, :2], sinks, at), (q[..., :32], sinks, at), (q, sinks.float(), at), (q, sinks[:11], at),
                         (q, sinks, at.float()), (q, sinks, at.expand(3)), (q, sinks, at[0]), (q, sinks.view(3, 4), at)):
        with pytest.raises(AssertionError):
            T.mxfp4_attention(qq, cache, s, 1.0, 0, start)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(RuntimeError, match="sm_scale"):
            T.mxfp4_attention(q, cache, sinks, scale, 0, at)
    for window in (-1, -(2**32) + 5):
        with pytest.raises(RuntimeError, match="window"):
            T.mxfp4_attention(q, cache, sinks, 1.0, window, at)
    with pytest.raises(RuntimeError, match="query heads"):
        T.mxfp4_attention(q.repeat(1, 1, 1, 20, 1), cache, None, 1.0, 0, at)
    with pytest.raises(NotImplementedError):
        T.mxfp4_attention(torch.zeros(2, 1, 3, 4, 128, dtype=torch.bfloat16, device="cuda"), T.mxfp4_cache(2, 10, 3, 128), None, 1.0, 0, at)
    with pytest.raises(AssertionError, match="one token"):
        T.mxfp4_attention_decode(q.expand(2, 2, 3, 4, 64), cache, None, 1.0, 0, at)
    with pytest.raises(RuntimeError, match="GPU"):
        T.mxfp4_attention(q, cache, sinks.cpu(), 1.0, 0, at)


@gpu
def test_more_heads_and_values_than_32_bits_count():
    """Numbers of heads and of blocks that are 8 and 2 beyond a power of two: refused, not taken for 8 heads of 64."""
    cache = T.Mxfp4Cache(*(t[:, :, :1].expand(1, 4, 2**32 + 8, *t.shape[3:]) for t in T.mxfp4_cache(1, 4, 1)))
    blocks, scales = torch.empty(1, 1, 1, 2**27 + 2, 16, dtype=torch.uint8, device="cuda"), torch.empty(1, 1, 1, 2**27 + 2, dtype=torch.uint8, device="cuda")
    for bad, what in ((cache, "heads"), (T.Mxfp4Cache(blocks, scales, blocks, scales), "head_dim")):
        with pytest.raises(AssertionError, match=what):
            T.mxfp4_cache_read(bad)
    del blocks, scales, bad
    torch.cuda.empty_cache()
