"""MXFP4 quantisation and products, routing to experts and the experts' two products against their definitions in float64 on the
CPU. Tolerances: products of bf16 (or MXFP4) values are exact in fp32, so a sum of K of them is off by at most K 2^-23 of the sum of
their magnitudes however it is ordered, and a bf16 result by 2^-8 of itself (half a place, doubled for the binade's edge)."""
import ctypes as C
import math

import pytest
import torch

import tritonllm_amd as T
from tritonllm_amd import _lib

gpu = pytest.mark.gpu
FP4 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
ALPHA, LIMIT = 1.702, 7.0


def values(blocks, scales):
    """MXFP4 in float64; a scale byte of 255 is NaN."""
    v = torch.stack((FP4[(blocks & 15).long()], FP4[(blocks >> 4).long()]), -1).flatten(-2)
    p = torch.ldexp(torch.ones((), dtype=torch.float64), scales.long() - 127)
    return (v * torch.where(scales == 255, math.nan, p)[..., None]).flatten(-2)


def random_mx(g, *shape, lo=118, hi=123):
    *rows, k = shape
    return (torch.randint(0, 256, (*rows, k // 32, 16), generator=g, dtype=torch.uint8),
            torch.randint(lo, hi, (*rows, k // 32), generator=g, dtype=torch.uint8))


def cuda(*ts):
    return [t if t is None else t.cuda() for t in ts]


def check_product(got, want, magnitude, k, what=""):
    """got bf16 / want float64 / the sum of the products' magnitudes"""
    got = got.double().cpu()
    assert got.shape == want.shape
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan), what
    off = (got - want).abs()
    ok = nan | (off <= 2.0**-8 * want.abs() + k * 2.0**-23 * magnitude) | (got == want)
    assert ok.all(), f"{what}: {(~ok).sum()} of {ok.numel()} off, the worst {off[~ok].max()}"


# ---- quantisation -----------------------------------------------------------------------------------------------------------
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
    scale = torch.where(bad, 255, (e + 127).long()).to(torch.uint8)
    code = code.to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(32,), (1, 64), (3, 96), (17, 2880), (2, 5, 160), (257, 4096)])
def test_quantize(dtype, shape):
    g = torch.Generator().manual_seed(len(shape) * 100 + shape[-1])
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-12, 12, shape, generator=g).float() * (torch.rand(shape, generator=g) < 0.1))
    x = x.to(dtype)
    blocks, scales = T.mxfp4_quantize(x.cuda())
    want_b, want_s = quantize_ref(x)
    assert blocks.shape == (*shape[:-1], shape[-1] // 32, 16) and scales.shape == blocks.shape[:-1]
    assert torch.equal(scales.cpu(), want_s) and torch.equal(blocks.cpu(), want_b)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_edges(dtype):
    """Ties, saturation, zeros of both signs, subnormals, the type's largest, and blocks with NaN or infinity beside fine ones."""
    info = torch.finfo(dtype)
    x = torch.zeros(14, 32, dtype=torch.float64)
    x[0] = torch.arange(32) / 4                                    # scale 2^0: every midpoint of the codes
    x[1] = -torch.arange(32) / 4
    x[2, 3] = 7.9                                                  # beyond 6: saturates
    x[3] = -0.0
    x[4, 5] = info.tiny
    x[5] = info.smallest_normal * torch.arange(32) / 32            # subnormals (and the smallest normal's neighbours)
    x[6, 0] = info.max
    x[7, 31] = -info.max
    x[8, 2] = math.nan
    x[9, 2] = math.inf
    x[10, 2] = -math.inf
    x[11] = info.smallest_normal * torch.arange(32)
    x[12, ::2] = 1.0
    x[13] = torch.linspace(-1, 1, 32, dtype=torch.float64)
    x = x.to(dtype)
    blocks, scales = T.mxfp4_quantize(x.cuda())
    want_b, want_s = quantize_ref(x)
    assert torch.equal(scales.cpu(), want_s)
    assert torch.equal(blocks.cpu(), want_b)
    assert scales[8:11].eq(255).all() and blocks[8:11].eq(0).all()


@gpu
def test_quantize_strides():
    x = torch.randn(9, 400, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    for view in (x[:, 8:360], x[:, 1:33], x[::2, :64], x.t()[:, :1].expand(400, 32), x[:0, :32], x[:, :0]):
        blocks, scales = T.mxfp4_quantize(view)
        want_b, want_s = quantize_ref(view.cpu().contiguous()) if view.numel() else (blocks.cpu(), scales.cpu())
        assert torch.equal(blocks.cpu(), want_b) and torch.equal(scales.cpu(), want_s)
    odd = torch.empty(33 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(33, 64).copy_(x.flatten()[: 33 * 64].view(33, 64))   # 2 bytes off
    assert torch.equal(T.mxfp4_quantize(odd)[0].cpu(), quantize_ref(odd.cpu())[0])


@gpu
def test_quantized_values_come_back():
    """What is in MXFP4 already stays as it is."""
    g = torch.Generator().manual_seed(8)
    blocks, scales = random_mx(g, 40, 320, lo=100, hi=140)
    blocks[..., 0] = 7                                             # (a 6 in every block: its scale is the largest that holds it)
    x = values(blocks, scales).float().cuda()
    again, s = T.mxfp4_quantize(x)
    assert torch.equal(s.cpu(), scales) and torch.equal(values(again.cpu(), s.cpu()).float(), x.cpu())


# ---- the product ------------------------------------------------------------------------------------------------------------
def linear_case(rows, n, k, acts, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed + rows * 7 + n * 3 + k)
    w, ws = random_mx(g, n, k)
    b = torch.randn(n, generator=g).bfloat16() if bias else None
    if acts == "bf16":
        x, xs = torch.randn(rows, k, generator=g).bfloat16(), None
        xv = x.double()
    else:
        x, xs = random_mx(g, rows, k, lo=123, hi=128)
        xv = values(x, xs)
    wv = values(w, ws)
    want, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    if bias:
        want, mag = want + b.double(), mag + b.double().abs()
    return x, xs, w, ws, b, want, mag


# (the last: long rows, and sizes that fill whole tiles of each shape)
LINEAR = [(3, 40, 20480), (17, 70, 40960), (300, 33, 40960), (300, 64, 8192), (2100, 2000, 96), (1, 2880, 4096), (1, 16, 32), (2, 1, 64), (3, 15, 96), (5, 17, 160), (16, 33, 224), (17, 127, 288), (31, 64, 2880), (33, 130, 512),
          (65, 257, 608), (100, 100, 1024), (129, 320, 736), (200, 29, 2048), (257, 511, 352), (300, 640, 2880), (515, 1100, 160)]


@gpu
@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
@pytest.mark.parametrize("rows,n,k", LINEAR)
def test_linear(rows, n, k, acts):
    x, xs, w, ws, b, want, mag = linear_case(rows, n, k, acts)
    dx, dxs, dw, dws, db = cuda(x, xs, w, ws, b)
    check_product(T.mxfp4_linear(dx, dw, dws, db, x_scales=dxs), want, mag, k)


@gpu
@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
@pytest.mark.parametrize("rows", [1, 20, 300])
def test_linear_without_bias_and_odd_shapes(rows, acts):
    x, xs, w, ws, b, want, mag = linear_case(rows, 48, 320, acts, bias=False)
    dx, dxs, dw, dws = cuda(x, xs, w, ws)
    got = T.mxfp4_linear(dx, dw, dws, x_scales=dxs)
    check_product(got, want, mag, 320)
    lead = (2, rows // 2) if rows % 2 == 0 else (1, 1, rows)
    more = T.mxfp4_linear(dx.reshape(*lead, *dx.shape[1:]), dw, dws, x_scales=None if xs is None else dxs.reshape(*lead, -1))
    assert torch.equal(more.reshape(rows, -1), got)
    assert T.mxfp4_linear(dx[:0], dw, dws, x_scales=None if xs is None else dxs[:0]).shape == (0, 48)
    if acts == "bf16":
        wide = torch.randn(rows, 400).bfloat16().cuda()
        for at in (8, 3):                                          # aligned rows of a wider matrix, and rows that have to be copied
            wide[:, at: at + 320] = dx
            assert torch.equal(T.mxfp4_linear(wide[:, at: at + 320], dw, dws), got)


@gpu
@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_linear_special_values(rows, acts):
    """NaN blocks of the weight spoil their output alone, NaN and infinite activations their row; the smallest and largest scales count."""
    x, xs, w, ws, b, _, _ = linear_case(rows, 70, 224, acts)
    ws[3, 2] = 255
    ws[69, 6] = 255
    ws[5], ws[6] = 0, 1
    ws[7] = 230
    if acts == "bf16":
        x[0, 100] = math.nan
        if rows > 20:
            x[17, 223] = math.inf
            w[:, 6, 15] |= 0x10                                    # (no weight there is 0)
        xv = x.double()
    else:
        xs[0, 3] = 255
        if rows > 20:
            xs[17] = 0
        xv = values(x, xs)
    wv = values(w, ws)
    want = torch.stack([(xv * wv[i]).sum(1) for i in range(70)], 1) + b.double()
    mag = (xv.abs()[:, None] * wv.abs()).sum(2).nan_to_num(0, 0, 0) + b.double().abs()
    dx, dxs, dw, dws, db = cuda(x, xs, w, ws, b)
    got = T.mxfp4_linear(dx, dw, dws, db, x_scales=dxs)
    check_product(got, want, mag, 224)


@gpu
@pytest.mark.parametrize("rows,n,k", [(2048, 4096, 1024), (2048, 5120, 1024), (1000, 2880, 2048), (700, 2880, 5120), (2048, 5120, 2880), (129, 200, 2880),
                                      (520, 5001, 2880), (330, 8000, 96), (3000, 1100, 160)])
@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
def test_linear_of_prompts(rows, n, k, acts):
    """The larger tiles; the reference is a float64 product on the GPU."""
    g = torch.Generator().manual_seed(rows + n + k)
    (w, ws), b = random_mx(g, n, k), torch.randn(n, generator=g).bfloat16()
    x, xs = (torch.randn(rows, k, generator=g).bfloat16(), None) if acts == "bf16" else random_mx(g, rows, k, lo=123, hi=128)
    xv, wv = (x.double() if xs is None else values(x, xs)).cuda(), values(w, ws).cuda()
    want, mag = (xv @ wv.t()).cpu() + b.double(), (xv.abs() @ wv.abs().t()).cpu() + b.double().abs()
    dx, dxs, dw, dws, db = cuda(x, xs, w, ws, b)
    check_product(T.mxfp4_linear(dx, dw, dws, db, x_scales=dxs), want, mag, k)


# Sizes by the kernels that take them, few rows: 16, 32 and 64 weight rows to a workgroup, with 1 - 4, 5 - 8 and up to 16 rows in the last
# run of rows; and the tiles, with edges in both directions.
STREAMS = [(16, 100, 352), (23, 90, 736), (40, 1500, 96), (3, 4200, 288), (7, 4130, 224), (12, 4160, 736), (64, 5120, 2880), (20, 9001, 1056), (33, 8200, 96),
           (190, 2500, 160), (130, 3333, 416), (25, 32770, 64), (22, 16388, 224)]
TILES = [(1900, 4801, 1312), (1025, 4800, 2880), (2600, 4321, 1120), (2333, 5100, 480)]


def linear_on_gpu(x, xs, w, ws, b):
    """float64 on the GPU: the product, the magnitudes"""
    v = lambda t, s: values(t, s).cuda()
    xv, wv = x.double().cuda() if xs is None else v(x, xs), v(w, ws)
    add = torch.zeros((), dtype=torch.float64) if b is None else b.double()
    return (xv @ wv.t()).cpu() + add, (xv.abs().nan_to_num(0, 0, 0) @ wv.abs().nan_to_num(0, 0, 0).t()).cpu() + add.abs()


@gpu
@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
@pytest.mark.parametrize("rows,n,k", STREAMS + TILES)
def test_linear_of_each_kernel(rows, n, k, acts):
    """NaN blocks of the weight and NaN rows among the others, and rows of a wider matrix."""
    g = torch.Generator().manual_seed(rows + n + k)
    (w, ws), b = random_mx(g, n, k), torch.randn(n, generator=g).bfloat16()
    x, xs = (torch.randn(rows, k, generator=g).bfloat16(), None) if acts == "bf16" else random_mx(g, rows, k, lo=123, hi=128)
    for i in (0, n // 2, n - 1):
        ws[i, (i * 5 + k // 32 - 1) % (k // 32)] = 255
    bad = rows - 1 - rows // 3
    if acts == "bf16":
        x[bad, k - 1] = math.nan
    else:
        xs[bad, -1] = 255
    want, mag = linear_on_gpu(x, xs, w, ws, b)
    assert want[bad].isnan().all() and want.isnan().sum() == n + 3 * rows - 3
    dx, dxs, dw, dws, db = cuda(x, xs, w, ws, b)
    got = T.mxfp4_linear(dx, dw, dws, db, x_scales=dxs)
    check_product(got, want, mag, k)
    if acts == "bf16":
        wide = torch.full((rows, k + 24), math.nan, dtype=torch.bfloat16, device="cuda")
        wide[:, 8: 8 + k] = dx
        assert torch.equal(T.mxfp4_linear(wide[:, 8: 8 + k], dw, dws, db).view(torch.int16), got.view(torch.int16))


@gpu
@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
@pytest.mark.parametrize("rows,n", [(1, 70), (40, 1500), (33, 8200), (16, 100), (300, 70), (700, 5000), (1900, 4800), (2333, 5100)])
def test_linear_with_the_smallest_and_largest_scales(rows, n, acts):
    """Weights down to 2^-128 (subnormal in bf16) and up to the last scale bytes, with activations that bring the sums back, and nothing
    beside them. Values of 2^128 and more are infinite beside bf16 activations, and as they are beside MXFP4 ones."""
    g = torch.Generator().manual_seed(rows + n)
    k = 224
    for at, lo, hi in ((100, 0, 4), (-110, 250, 253), (-110, 253, 255)):
        w, ws = random_mx(g, n, k, lo=lo, hi=hi)
        if acts == "bf16":
            x, xs = (torch.randn(rows, k, generator=g).bfloat16().float() * 2.0**at).bfloat16(), None
            xv = x.double()
        else:
            x, xs = random_mx(g, rows, k, lo=127 + at, hi=130 + at)
            xv = values(x, xs)
        wv = values(w, ws)
        if acts == "bf16":
            wv = torch.where(wv.abs() >= 2.0**128, torch.sign(wv) * math.inf, wv)
        want = (xv.cuda() @ wv.cuda().t()).cpu()
        mag = (xv.abs().cuda() @ wv.abs().nan_to_num(0, 0, 0).cuda().t()).cpu().nan_to_num(0, 0, 0)
        assert (want[want.isfinite()].abs() < 2.0**60).all() and (hi < 255 or acts == "mxfp4") == bool(want.isfinite().all())
        if hi < 255 or acts == "mxfp4":
            assert want.abs().median() > 2.0**-60
        dx, dxs, dw, dws = cuda(x, xs, w, ws)
        check_product(T.mxfp4_linear(dx, dw, dws, x_scales=dxs), want, mag, k, f"scales from {lo}")


@gpu
@pytest.mark.parametrize("rows", [5, 300])
def test_linear_of_unaligned_views(rows):
    """Weights, scales and activations that begin anywhere are copied, or read as they are where that is possible."""
    x, _, w, ws, b, want, mag = linear_case(rows, 61, 288, "bf16")
    dx, dw, dws, db = cuda(x, w, ws, b)
    big_w, big_s = torch.zeros(70, 9, 16, dtype=torch.uint8, device="cuda"), torch.zeros(70, 9, dtype=torch.uint8, device="cuda")
    for at in (1, 5):
        big_w[at: at + 61], big_s[at: at + 61] = dw, dws
        check_product(T.mxfp4_linear(dx, big_w[at: at + 61], big_s[at: at + 61], db), want, mag, 288)
    wide = torch.zeros(61, 12, 16, dtype=torch.uint8, device="cuda")
    wide[:, 2:11] = dw
    check_product(T.mxfp4_linear(dx.t().contiguous().t(), wide[:, 2:11], dws, db), want, mag, 288)


@gpu
@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
def test_linear_of_rows_beyond_32_bits(acts):
    """Activations of more than 4 GiB: the first rows, ones from the middle and the last."""
    rows, k, n = ((1 << 22) + 133, 512, 16) if acts == "bf16" else ((1 << 23) + 133, 1024, 16)
    g = torch.Generator(device="cuda").manual_seed(1)
    w, ws = random_mx(torch.Generator().manual_seed(2), n, k)
    if acts == "bf16":
        x, xs = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda").normal_(generator=g), None
    else:
        x = torch.randint(0, 256, (rows, k // 32, 16), generator=g, dtype=torch.uint8, device="cuda")
        xs = torch.randint(120, 130, (rows, k // 32), generator=g, dtype=torch.uint8, device="cuda")
    assert x.numel() * x.element_size() > 1 << 32
    got = T.mxfp4_linear(x, *cuda(w, ws), x_scales=xs)
    wv = values(w, ws)
    for first in (0, rows // 2, rows - 300):
        part = slice(first, first + 300)
        xv = x[part].cpu().double() if xs is None else values(x[part].cpu(), xs[part].cpu())
        check_product(got[part], xv @ wv.t(), xv.abs() @ wv.abs().t(), k, f"rows from {first} on")


@gpu
def test_quantize_then_linear_is_the_product_of_the_values():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(77, 2880, generator=g).bfloat16()
    w, ws = random_mx(g, 96, 2880)
    xq, xs = T.mxfp4_quantize(x.cuda())
    xv, wv = values(xq.cpu(), xs.cpu()), values(w, ws)
    check_product(T.mxfp4_linear(xq, w.cuda(), ws.cuda(), x_scales=xs), xv @ wv.t(), xv.abs() @ wv.abs().t(), 2880)


# ---- routing ----------------------------------------------------------------------------------------------------------------
def route_ref(logits, top, score="softmax", bias=None, groups=1, kept=1, renorm=True, scale=1.0):
    """In float64 and in plain loops over the choices; also how near the nearest choice that could go either way was."""
    z = logits.double().clone()
    z[z.isnan()] = -math.inf
    tokens, n = z.shape
    if score == "softmax":
        m = z.amax(1, keepdim=True)
        s = torch.where(z == -math.inf, 0.0, torch.where(z == m, 1.0, torch.exp(z - m.clamp(min=-1e300, max=1e300))))
        s = s / s.sum(1, keepdim=True).clamp(min=1e-300)
    else:
        s = 1 / (1 + torch.exp(-z))
    c = z.clone() if bias is None else s + bias.double()
    c[c.isnan()] = -math.inf
    near = torch.full((tokens,), math.inf, dtype=torch.float64)
    if groups > 1:
        by = (s if bias is None else c).view(tokens, groups, -1)
        v = by.sort(2, descending=True).values[..., :2].sum(2)
        o = torch.sort(v, dim=1, descending=True, stable=True)
        if kept < groups:
            near = torch.minimum(near, o.values[:, kept - 1] - o.values[:, kept])
        keep = torch.zeros(tokens, groups, dtype=torch.bool).scatter_(1, o.indices[:, :kept], True)
        out = ~keep.repeat_interleave(n // groups, 1)
    else:
        out = torch.zeros(tokens, n, dtype=torch.bool)
    order = torch.empty(tokens, n, dtype=torch.long)
    if tokens > 5000:                                              # (loops take too long there)
        order = torch.sort(torch.where(out, -math.inf, c), dim=1, descending=True, stable=True).indices
    for t in range(tokens if tokens <= 5000 else 0):
        order[t] = torch.tensor(sorted(range(n), key=lambda e: (bool(out[t, e]), -c[t, e].item(), e)))
    best = order[:, : min(top + 1, n)]
    if bias is not None and best.shape[1] > 1:
        gaps = -(c.gather(1, best).diff(dim=1))
        same = (z.gather(1, best).diff(dim=1) == 0) & (bias.double()[best].diff(dim=1) == 0)    # equal in any precision
        near = torch.minimum(near, torch.where(same | out.gather(1, best[:, 1:]), math.inf, gaps).amin(1))
    best = best[:, :top]
    w = s.gather(1, best)
    if renorm:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
    return best, w * scale, near


def check_plan(r, tokens, experts, top):
    flat = r.experts.reshape(-1).cpu().long()
    assert r.experts.dtype == r.order.dtype == r.offsets.dtype == torch.int32 and r.weights.dtype == torch.float32
    assert torch.equal(r.order.cpu().long(), torch.sort(flat, stable=True).indices)
    want = torch.zeros(experts + 1, dtype=torch.long)
    want[1:] = torch.bincount(flat, minlength=experts).cumsum(0)
    assert torch.equal(r.offsets.cpu().long(), want)


def check_route(logits, top, near_at_least=1e-5, **how):
    named = dict(score=how.get("score", "softmax"), bias=how.get("bias"), groups=how.get("groups", 1), kept=how.get("kept", 1),
                 renorm=how.get("renorm", True), scale=how.get("scale", 1.0))
    best, w, near = route_ref(logits, top, **named)
    r = T.moe_route(logits.cuda(), top, score=named["score"], bias=None if named["bias"] is None else named["bias"].cuda(), n_groups=named["groups"],
                    topk_groups=named["kept"], renormalize=named["renorm"], scale=named["scale"])
    sure = near > near_at_least                                    # the others hang on fp32's last places
    assert sure.double().mean() > 0.9
    assert torch.equal(r.experts.cpu().long()[sure], best[sure])
    torch.testing.assert_close(r.weights.cpu().double()[sure], w[sure], rtol=2e-6, atol=1e-7 * abs(named["scale"]))
    check_plan(r, logits.shape[0], logits.shape[1], top)
    return r


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,experts,top", [(1, 1, 1), (1, 32, 4), (8, 32, 4), (7, 5, 5), (63, 64, 8), (64, 65, 3), (65, 33, 2), (200, 128, 4), (300, 257, 8),
                                                (129, 512, 32), (1000, 32, 4), (4097, 17, 2), (6001, 32, 4),
                                                (6003, 17, 16), (8191, 256, 8), (6500, 500, 5), (9000, 100, 1), (6100, 64, 17)])
def test_route(tokens, experts, top, dtype):
    g = torch.Generator().manual_seed(tokens + experts)
    logits = (1.5 * torch.randn(tokens, experts, generator=g)).to(dtype)
    check_route(logits, top)
    check_route(logits, top, score="sigmoid", renorm=False, scale=2.5)


@gpu
@pytest.mark.parametrize("tokens,experts,top,groups,kept", [(1, 16, 2, 4, 2), (33, 256, 8, 8, 4), (70, 48, 6, 3, 2), (150, 512, 8, 64, 8), (90, 160, 6, 8, 3), (66, 8, 1, 8, 1),
                                                            (500, 64, 8, 2, 1), (6002, 256, 8, 8, 4), (6100, 64, 4, 8, 3), (6050, 60, 6, 5, 2), (7000, 512, 16, 16, 5)])
def test_route_groups(tokens, experts, top, groups, kept):
    g = torch.Generator().manual_seed(tokens * experts)
    logits = (1.5 * torch.randn(tokens, experts, generator=g)).bfloat16()
    bias = 0.1 * torch.randn(experts, generator=g)
    check_route(logits, top, score="sigmoid", bias=bias, groups=groups, kept=kept, scale=1.5)
    check_route(logits, top, score="sigmoid", groups=groups, kept=kept)
    check_route(logits, top, score="softmax", groups=groups, kept=kept, near_at_least=1e-7)
    check_route(logits, top, score="softmax", bias=bias)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,experts,top", [(1, 512, 8), (64, 300, 32), (17, 512, 8), (33, 257, 5), (9, 200, 3)])
def test_route_of_few_tokens_to_many_experts(tokens, experts, top, dtype):
    g = torch.Generator().manual_seed(tokens + experts + 1)
    logits = (1.5 * torch.randn(tokens, experts, generator=g)).to(dtype)
    bias = 0.5 * torch.randn(experts, generator=g)
    check_route(logits, top)
    check_route(logits, top, score="sigmoid", renorm=False, scale=2.5)
    for groups, kept in ((64, 9), (8, 4)):
        if experts % groups == 0:
            check_route(logits, top, score="sigmoid", bias=bias, groups=groups, kept=kept)
            check_route(logits, top, groups=groups, kept=kept, near_at_least=1e-7)


@gpu
@pytest.mark.parametrize("tokens", [5, 100, 6500])
def test_route_ties_and_masks(tokens):
    """Equal logits go to the lowest index; -inf, NaN and rows of nothing else; the lowest finite value is no mask."""
    g = torch.Generator().manual_seed(tokens)
    logits = torch.randint(-2, 3, (tokens, 40), generator=g).float()
    check_route(logits, 6)
    check_route(logits, 6, score="sigmoid")
    logits[0] = 1.0
    logits[1, 3:] = -math.inf                                      # three are left for six places
    logits[2, ::2] = math.nan
    logits[3] = -math.inf
    logits[4] = torch.finfo(torch.float32).min
    for score in ("softmax", "sigmoid"):
        r = check_route(logits, 6, score=score)
        assert r.experts[0].tolist() == list(range(6)) == r.experts[3].tolist()
        assert r.weights[3].eq(0).all() and r.weights[1, 3:].eq(0).all() and r.weights.isfinite().all()
    lowest = T.moe_route(logits.cuda(), 6).weights[4]
    assert (lowest == lowest[0]).all() and lowest[0] > 0.1
    inf = logits.clone()
    inf[0, 7] = math.inf
    r = T.moe_route(inf.cuda(), 2)
    assert r.experts[0].tolist() == [7, 0] and r.weights[0].tolist() == [1.0, 0.0]


@gpu
def test_route_shapes():
    r = T.moe_route(torch.empty(0, 32, device="cuda"), 4)
    assert r.experts.shape == r.weights.shape == (0, 4) and r.order.shape == (0,) and r.offsets.tolist() == [0] * 33
    x = torch.randn(6, 50, generator=torch.Generator().manual_seed(1))
    want = T.moe_route(x[:, :32].contiguous().cuda(), 4)
    for view in (x.cuda()[:, :32], x.cuda().t().contiguous().t()[:, :32], x[:, :32].reshape(2, 3, 32).cuda()):
        for a, b in zip(T.moe_route(view, 4), want):
            assert torch.equal(a, b)


# ---- the experts ------------------------------------------------------------------------------------------------------------
def plan_of(chosen, experts):
    flat = chosen.reshape(-1).long()
    offsets = torch.zeros(experts + 1, dtype=torch.int32)
    offsets[1:] = torch.bincount(flat, minlength=experts).cumsum(0).int()
    return torch.sort(flat, stable=True).indices.int(), offsets


def experts_case(tokens, experts, top, hidden, inner, seed=0, spread=1.0):
    """Routing (uneven with a small spread: some experts get nothing, few most) and both weights."""
    g = torch.Generator().manual_seed(seed + tokens * 31 + experts)
    favour = torch.randn(experts, generator=g) * 2 / spread
    chosen = (torch.randn(tokens, experts, generator=g) + favour).topk(top, 1).indices.int()
    weights = torch.softmax(torch.randn(tokens, top, generator=g), 1)
    order, offsets = plan_of(chosen, experts)
    return g, T.MoeRouting(chosen, weights, order, offsets), random_mx(g, experts, 2 * inner, hidden), random_mx(g, experts, hidden, inner)


def by_expert(x, routing, w, ws, bias):
    """rows in the plan's order -> (sums, magnitudes), float64"""
    y = torch.empty(len(routing.order), w.shape[1], dtype=torch.float64)
    m = torch.empty_like(y)
    for e in range(w.shape[0]):
        lo, hi = routing.offsets[e], routing.offsets[e + 1]
        wv = values(w[e], ws[e])
        y[lo:hi], m[lo:hi] = x[lo:hi] @ wv.t(), x[lo:hi].abs() @ wv.abs().t()
        if bias is not None:
            y[lo:hi] += bias[e].double()
            m[lo:hi] += bias[e].double().abs()
    return y, m


EXPERTS = [(1, 4, 1, 32, 32), (1, 32, 4, 2880, 96), (2, 8, 2, 64, 160), (7, 8, 8, 96, 64), (8, 32, 4, 224, 352), (33, 17, 3, 160, 32), (40, 4, 2, 480, 96),
           (3000, 2, 2, 96, 352), (3000, 2, 2, 704, 64), (1000, 32, 4, 64, 544), (1000, 32, 4, 1088, 64), (64, 8, 4, 128, 288), (150, 3, 2, 352, 64), (300, 8, 3, 288, 160), (700, 2, 1, 64, 128), (257, 64, 4, 96, 96), (1000, 5, 4, 32, 32)]


@gpu
@pytest.mark.parametrize("limit,bias", [(7.0, True), (None, False)])
@pytest.mark.parametrize("tokens,experts,top,hidden,inner", EXPERTS)
def test_mlp1(tokens, experts, top, hidden, inner, limit, bias):
    g, routing, (w, ws), _ = experts_case(tokens, experts, top, hidden, inner)
    x = torch.randn(tokens, hidden, generator=g).bfloat16()
    b = torch.randn(experts, 2 * inner, generator=g).bfloat16() if bias else None
    y, m = by_expert(x.double()[(routing.order // top).long()], routing, w, ws, b)
    off = hidden * 2.0**-23 * m
    lim = math.inf if limit is None else limit
    gate, lin = y[:, 0::2].clamp(max=lim), y[:, 1::2].clamp(-lim, lim)
    want = gate * torch.sigmoid(ALPHA * gate) * (lin + 1)
    # of g sigmoid(a g): the slope is at most 1.1; fp32's exp, division and products add a few of its places
    room = 2.0**-8 * want.abs() + 1.1 * (lin + 1).abs() * off[:, 0::2] + gate.abs() * off[:, 1::2] + 1e-5 * want.abs() + 1e-30
    got = T.moe_mlp1(x.cuda(), T.MoeRouting(*cuda(*routing)), *cuda(w, ws, b), alpha=ALPHA, limit=limit)
    assert got.shape == want.shape and got.dtype == torch.bfloat16
    d = (got.double().cpu() - want).abs()
    assert (d <= room).all(), f"{(d > room).sum()} of {d.numel()} off, the worst {(d / room).max()} of the room"


@gpu
@pytest.mark.parametrize("residual,bias", [(True, True), (False, False)])
@pytest.mark.parametrize("tokens,experts,top,hidden,inner", EXPERTS)
def test_mlp2(tokens, experts, top, hidden, inner, residual, bias):
    g, routing, _, (w, ws) = experts_case(tokens, experts, top, hidden, inner)
    h = torch.randn(tokens * top, inner, generator=g).bfloat16()
    b = torch.randn(experts, hidden, generator=g).bfloat16() if bias else None
    res = torch.randn(tokens, hidden, generator=g).bfloat16() if residual else None
    y, m = by_expert(h.double(), routing, w, ws, b)
    wt = routing.weights.double().reshape(-1)[routing.order.long()][:, None]
    token = (routing.order // top).long()
    want = torch.zeros(tokens, hidden, dtype=torch.float64).index_add_(0, token, y * wt)
    mag = torch.zeros_like(want).index_add_(0, token, m * wt)
    if residual:
        want, mag = want + res.double(), mag + res.double().abs()
    dr = T.MoeRouting(*cuda(*routing))
    dh, dw, dws, db, dres = cuda(h, w, ws, b, res)
    got = T.moe_mlp2(dh, dr, dw, dws, db, residual=dres)
    check_product(got, want, mag, inner + top)
    assert torch.equal(T.moe_mlp2(dh, dr, dw, dws, db, residual=dres), got)      # the same order of sums every time
    if residual:
        assert T.moe_mlp2(dh, dr, dw, dws, db, residual=dres, out=dres) is dres and torch.equal(dres, got)


COUNTS = [1, 3, 4, 5, 8, 9, 16, 17, 40, 0, 33]                     # tokens of each expert: every number of rows that the weight streams past


def by_expert_on_gpu(x, routing, w, ws, bias):
    y, m = [], []
    for e in range(w.shape[0]):
        rows = x[routing.offsets[e]: routing.offsets[e + 1]].cuda()
        wv, b = values(w[e], ws[e]).cuda(), bias[e].double().cuda()
        y.append(rows @ wv.t() + b)
        m.append(rows.abs() @ wv.abs().nan_to_num(0, 0, 0).t() + b.abs())
    return torch.cat(y).cpu(), torch.cat(m).cpu()


@gpu
@pytest.mark.parametrize("n", [100, 500, 1730, 4160])
@pytest.mark.parametrize("k", [160, 1056])
@pytest.mark.parametrize("scale", [1, 3])
def test_experts_of_each_number_of_rows(n, k, scale):
    """Experts of none, one and up to forty tokens (or three times as many, in tiles) at each width of a workgroup; a NaN block in one expert's weight."""
    counts = [c * scale for c in COUNTS]
    tokens, experts = sum(counts), len(counts)
    g = torch.Generator().manual_seed(n + k + scale)
    chosen = torch.repeat_interleave(torch.arange(experts), torch.tensor(counts))[torch.randperm(tokens, generator=g)].int()[:, None]
    routing = T.MoeRouting(chosen, torch.rand(tokens, 1, generator=g) + 0.1, *plan_of(chosen, experts))
    w, ws = random_mx(g, experts, n, k)
    ws[7, n - 1, k // 32 - 1] = 255
    b = torch.randn(experts, n, generator=g).bfloat16()
    x = torch.randn(tokens, k, generator=g).bfloat16()
    dr = T.MoeRouting(*cuda(*routing))
    dx, dw, dws, db = cuda(x, w, ws, b)
    y, m = by_expert_on_gpu(x.double()[routing.order.long()], routing, w, ws, b)
    gate, lin = y[:, 0::2].clamp(max=LIMIT), y[:, 1::2].clamp(-LIMIT, LIMIT)
    want = gate * torch.sigmoid(ALPHA * gate) * (lin + 1)
    off = k * 2.0**-23 * m
    room = 2.0**-8 * want.abs() + 1.1 * (lin + 1).abs() * off[:, 0::2] + gate.abs() * off[:, 1::2] + 1e-5 * want.abs() + 1e-30
    got = T.moe_mlp1(dx, dr, dw, dws, db, alpha=ALPHA, limit=LIMIT).double().cpu()
    assert want.isnan().sum() == counts[7] and torch.equal(got.isnan(), want.isnan())
    assert ((got - want).abs() <= room)[~want.isnan()].all()
    y, m = by_expert_on_gpu(x.double(), routing, w, ws, b)
    wt = routing.weights.double()[routing.order.long()]
    at = routing.order.long()
    want, mag = torch.empty_like(y), torch.empty_like(m)
    want[at], mag[at] = y * wt, m * wt
    res = torch.randn(tokens, n, generator=g).bfloat16()
    check_product(T.moe_mlp2(dx, dr, dw, dws, db, residual=res.cuda()), want + res.double(), mag + res.double().abs(), k + 1)


@gpu
@pytest.mark.parametrize("tokens", [3, 200])
def test_experts_rows_from_strides_and_one_expert_for_all(tokens):
    g, _, (w, ws), (w2, ws2) = experts_case(tokens, 6, 2, 96, 64)
    chosen = torch.tensor([[5, 2]]).expand(tokens, 2).int().contiguous()
    routing = T.MoeRouting(*cuda(chosen, torch.full((tokens, 2), 0.5), *plan_of(chosen, 6)))
    wide = torch.randn(tokens, 200, generator=g).bfloat16().cuda()
    dense = T.moe_mlp1(wide[:, 8:104].contiguous(), routing, w.cuda(), ws.cuda())
    assert torch.equal(T.moe_mlp1(wide[:, 8:104], routing, w.cuda(), ws.cuda()), dense)
    wide[:, 101:197] = wide[:, 8:104].clone()
    assert torch.equal(T.moe_mlp1(wide[:, 101:197], routing, w.cuda(), ws.cuda()), dense)
    y, m = by_expert(dense.double().cpu(), T.MoeRouting(*[t.cpu() for t in routing]), w2, ws2, None)
    want = 0.5 * (y[:tokens] + y[tokens:])
    check_product(T.moe_mlp2(dense, routing, w2.cuda(), ws2.cuda()), want, 0.5 * (m[:tokens] + m[tokens:]), 66)


@gpu
def test_experts_nothing_to_do():
    g, routing, (w, ws), (w2, ws2) = experts_case(1, 4, 2, 64, 32)
    empty = T.moe_route(torch.empty(0, 4, device="cuda"), 2)
    h = T.moe_mlp1(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), empty, w.cuda(), ws.cuda())
    assert h.shape == (0, 32) and T.moe_mlp2(h, empty, w2.cuda(), ws2.cuda()).shape == (0, 64)


@gpu
def test_experts_nan_stays_with_its_token():
    tokens = 50
    g, routing, (w, ws), (w2, ws2) = experts_case(tokens, 6, 2, 96, 64)
    x = torch.randn(tokens, 96, generator=g).bfloat16()
    x[7, 5] = math.nan
    dr = T.MoeRouting(*cuda(*routing))
    h = T.moe_mlp1(x.cuda(), dr, w.cuda(), ws.cuda())
    bad = (routing.order // 2 == 7)
    assert h[bad.cuda()].isnan().all() and not h[~bad.cuda()].isnan().any()
    y = T.moe_mlp2(h, dr, w2.cuda(), ws2.cuda())
    assert y[7].isnan().all() and y.isnan().any(1).sum() == 1


def whole_case(g, n, k, *lead):
    """Weights of [..., n, k] that are multiples of a quarter, and rows' worth of them times -1, 0 and 1 exact in fp32 in any order
    (below 12 * 2^18, a multiple of 2^-2)."""
    return random_mx(g, *lead, n, k, lo=126, hi=129)


LONG = [229344, 229376, 262144]                                    # (whole blocks, the last an odd number of steps' worth; the longest rows)


@gpu
@pytest.mark.parametrize("acts", ["bf16", "mxfp4"])
@pytest.mark.parametrize("rows,n", [(1, 17), (5, 16), (17, 40), (220, 9)])
@pytest.mark.parametrize("k", LONG)
def test_linear_of_the_longest_rows(k, rows, n, acts):
    """All sums are exact: the result is the exact one, rounded once."""
    g = torch.Generator().manual_seed(k + rows)
    w, ws = whole_case(g, n, k)
    b = torch.randint(-9, 10, (n,), generator=g).bfloat16()
    x = torch.randint(-1, 2, (rows, k), generator=g).bfloat16().cuda()
    want = (x.double() @ values(w, ws).cuda().t() + b.cuda().double()).float().bfloat16()
    if acts == "mxfp4":
        x, xs = T.mxfp4_quantize(x)
        assert torch.equal(T.mxfp4_linear(x, *cuda(w, ws, b), x_scales=xs), want)
    else:
        assert torch.equal(T.mxfp4_linear(x, *cuda(w, ws, b)), want)


@gpu
@pytest.mark.parametrize("tokens", [1, 21, 120])
@pytest.mark.parametrize("k", LONG)
def test_experts_of_the_longest_rows(k, tokens):
    g = torch.Generator().manual_seed(k + tokens)
    chosen = torch.randint(0, 3, (tokens, 1), generator=g).int()
    chosen = torch.cat([chosen, (chosen + 1) % 3], 1)
    routing = T.MoeRouting(chosen, torch.full((tokens, 2), 0.5), *plan_of(chosen, 3))
    dr = T.MoeRouting(*cuda(*routing))
    w, ws = whole_case(g, 10, k, 3)
    b = torch.randint(-9, 10, (3, 10), generator=g).bfloat16()
    wv = values(w, ws).cuda()
    x = torch.randint(-1, 2, (tokens, k), generator=g).bfloat16().cuda()
    y = torch.einsum("tk,enk->ten", x.double(), wv) + b.cuda().double()
    pair = y.gather(1, chosen.cuda().long()[..., None].expand(-1, -1, 10))           # [tokens, 2, 10]
    rows = pair.reshape(-1, 10)[routing.order.cuda().long()]
    want = rows[:, 0::2] * torch.sigmoid(ALPHA * rows[:, 0::2]) * (rows[:, 1::2] + 1)
    got = T.moe_mlp1(x, dr, *cuda(w, ws, b), alpha=ALPHA, limit=None).double()
    assert ((got - want).abs() <= (2.0**-8 + 1e-5) * want.abs() + 1e-30).all()
    h = x.repeat_interleave(2, 0)[routing.order.cuda().long()]
    res = torch.randint(-9, 10, (tokens, 10), generator=g).bfloat16().cuda()
    want = (0.5 * (pair[:, 0] + pair[:, 1]) + res.double()).float().bfloat16()
    assert torch.equal(T.moe_mlp2(h, dr, *cuda(w, ws, b), residual=res), want)


@gpu
@pytest.mark.parametrize("tokens", [1, 9, 64, 65, 449])
@pytest.mark.parametrize("experts", [1, 5, 10, 16, 17, 32, 33, 48, 128])
@pytest.mark.parametrize("hidden", [96, 192, 2880])
def test_router_logits(tokens, experts, hidden):
    """Any number of experts, of any tokens."""
    g = torch.Generator().manual_seed(tokens + experts + hidden)
    x, w, b = torch.randn(tokens, hidden, generator=g).bfloat16(), torch.randn(experts, hidden, generator=g).bfloat16(), torch.randn(experts, generator=g).bfloat16()
    want, mag = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    dx, dw, db = cuda(x, w, b)
    check_product(T.router_logits(dx, dw, None), want, mag, hidden)
    check_product(T.router_logits(dx, dw, db), want + b.double(), mag + b.double().abs(), hidden)
    apart = torch.cat([x, x], 1)[:, hidden // 2 + 1: hidden // 2 + 1 + hidden]        # rows of a wider matrix, at any address
    v = apart.double()
    check_product(T.router_logits(torch.cat([dx, dx], 1)[:, hidden // 2 + 1: hidden // 2 + 1 + hidden], dw, db), v @ w.double().t() + b.double(),
                  v.abs() @ w.double().abs().t() + b.double().abs(), hidden)


@gpu
@pytest.mark.parametrize("tokens", [3, 70])
@pytest.mark.parametrize("experts,hidden", [(32, 192), (10, 192), (17, 192), (48, 96)])
def test_router_logits_of_operands_anywhere(tokens, experts, hidden):
    """Dense operands whose first value lies at any address."""
    g = torch.Generator().manual_seed(tokens + experts)
    ts = [torch.randn(shape, generator=g).bfloat16() for shape in ((tokens, hidden), (experts, hidden), (experts,))]
    x, w, b = (t.double() for t in ts)
    want, mag = x @ w.t() + b, x.abs() @ w.abs().t() + b.abs()
    for off in (1, 4):
        for which in range(3):
            d = cuda(*ts)
            d[which] = torch.zeros(d[which].numel() + off, dtype=torch.bfloat16, device="cuda")[off:].view(d[which].shape).copy_(d[which])
            assert d[which].is_contiguous() and d[which].data_ptr() % 16
            check_product(T.router_logits(*d), want, mag, hidden)


@gpu
@pytest.mark.parametrize("experts", [10, 16, 17])
def test_mlp_block_of_no_tokens(experts):
    m = mlp_block(experts=experts)
    x = torch.empty(0, 192, dtype=torch.bfloat16, device="cuda")
    assert T.router_logits(x, m.gate.weight, m.gate.bias).shape == (0, experts)
    assert m(x).shape == (0, 192) and m(x.view(2, 0, 192)).shape == (2, 0, 192)


@gpu
@pytest.mark.parametrize("hidden", [32, 33])
def test_router_logits_of_an_odd_number_for_many_tokens(hidden):
    tokens = 65535 + 70
    g = torch.Generator().manual_seed(hidden)
    x, w, b = torch.randn(tokens, hidden, generator=g).bfloat16(), torch.randn(3, hidden, generator=g).bfloat16(), torch.randn(3, generator=g).bfloat16()
    want, mag = x.double() @ w.double().t() + b.double(), x.double().abs() @ w.double().abs().t() + b.double().abs()
    check_product(T.router_logits(*cuda(x, w, b)), want, mag, hidden)


@gpu
@pytest.mark.parametrize("tokens", [3, 31, 250])
def test_rows_far_apart(tokens):
    """Rows that span almost 4 GiB are read where they lie; x of moe_mlp1 that spans more is refused."""
    g, routing, (w, ws), (w2, ws2) = experts_case(tokens, 4, 2, 288, 160)
    dr = T.MoeRouting(*cuda(*routing))
    dw, dws, dw2, dws2 = cuda(w, ws, w2, ws2)

    def far(rows, k, pitch):
        dense = torch.randn(rows, k, generator=g).bfloat16().cuda()
        return dense, torch.empty((rows - 1) * pitch + k, dtype=torch.bfloat16, device="cuda").as_strided((rows, k), (pitch, 1)).copy_(dense)

    most = ((1 << 31) - 2048) // (tokens - 1) // 8 * 8             # values between rows
    dense, x = far(tokens, 288, most)
    assert (tokens - 1) * most * 2 > 4000 << 20
    assert torch.equal(T.moe_mlp1(x, dr, dw, dws), T.moe_mlp1(dense, dr, dw, dws))
    assert torch.equal(T.mxfp4_linear(x, dw[0], dws[0]), T.mxfp4_linear(dense, dw[0], dws[0]))
    del x
    dense, x = far(tokens, 288, most + 2048)
    with pytest.raises(RuntimeError, match="4 GiB"):
        T.moe_mlp1(x, dr, dw, dws)
    del x
    dense, h = far(2 * tokens, 160, ((1 << 31) - 2048) // (2 * tokens - 1) // 8 * 8)
    assert torch.equal(T.moe_mlp2(h, dr, dw2, dws2), T.moe_mlp2(dense, dr, dw2, dws2))


# ---- together ---------------------------------------------------------------------------------------------------------------
def mlp_block(hidden=192, inner=160, experts=16, top=4, seed=0):
    g = torch.Generator().manual_seed(seed)
    m = T.MLPBlock(hidden, inner, experts, top, device="cuda")
    r = lambda *shape: (torch.randn(*shape, generator=g) / math.sqrt(shape[-1])).bfloat16()
    with torch.no_grad():
        m.norm.scale.copy_(1 + 0.1 * torch.randn(hidden, generator=g))
        m.gate.weight.copy_(3 * r(experts, hidden))
        m.gate.bias.copy_(r(experts))
        m.mlp1_bias.copy_(0.1 * torch.randn(experts, 2 * inner, generator=g))
        m.mlp2_bias.copy_(0.1 * torch.randn(experts, hidden, generator=g))
    return m.quantize_experts(r(experts, 2 * inner, hidden).cuda(), r(experts, hidden, inner).cuda())


def block_ref(m, x):
    """The block in float64, rounded to bf16 where one kernel hands over to the next; the routing is by its own logits."""
    bf = lambda v: v.bfloat16().double()
    t = x.double()
    t = bf(t * torch.rsqrt(t.square().mean(-1, keepdim=True) + m.norm.eps) * m.norm.scale.detach().cpu().double())
    logits = bf(t @ m.gate.weight.detach().cpu().double().t() + m.gate.bias.detach().cpu().double())
    v, e = torch.sort(logits, dim=1, descending=True, stable=True)
    top = m.experts_per_token
    sure = v[:, top - 1] - v[:, top] > 0.05                        # (a place of bf16 in a logit cannot change these tokens' experts)
    w = torch.softmax(v[:, :top], 1)
    w1, w2 = values(m.mlp1_blocks.cpu(), m.mlp1_scales.cpu()), values(m.mlp2_blocks.cpu(), m.mlp2_scales.cpu())
    out = x.double().clone()
    for i in range(len(x)):
        for j in range(top):
            k = e[i, j]
            y = w1[k] @ t[i] + m.mlp1_bias[k].detach().cpu().double()
            gate, lin = y[0::2].clamp(max=LIMIT), y[1::2].clamp(-LIMIT, LIMIT)
            h = bf(gate * torch.sigmoid(ALPHA * gate) * (lin + 1))
            out[i] += w[i, j] * (w2[k] @ h + m.mlp2_bias[k].detach().cpu().double())
    return out, sure


@gpu
@pytest.mark.parametrize("tokens,experts", [(1, 16), (7, 16), (70, 32), (300, 16), (9, 10)])
def test_mlp_block(tokens, experts):
    m = mlp_block(experts=experts)
    x = torch.randn(tokens, 192, generator=torch.Generator().manual_seed(tokens)).bfloat16()
    want, sure = block_ref(m, x)
    assert sure.double().mean() > 0.7 or tokens == 1
    got = m(x.cuda())
    # a place of bf16 in t, the logits and h each, and in the result: the kernels' tolerance here is twice the reference model's rounding
    torch.testing.assert_close(got.double().cpu()[sure], want[sure], rtol=2e-2, atol=2e-2)
    assert torch.equal(m(x.cuda().view(1, tokens, 192)).view(tokens, 192), got)


def gpt_oss_block(seed):
    """A block of gpt-oss's sizes: 32 experts, four to a token, 2880 wide."""
    m = T.MLPBlock(2880, 2880, 32, 4, device="cuda")
    g, d = torch.Generator().manual_seed(seed), torch.Generator(device="cuda").manual_seed(seed)
    with torch.no_grad():
        m.norm.scale.copy_(1 + 0.1 * torch.randn(2880, generator=g))
        m.gate.weight.copy_(3 * torch.randn(32, 2880, generator=g) / math.sqrt(2880))
        m.gate.bias.copy_(torch.randn(32, generator=g))
        m.mlp1_bias.copy_(0.1 * torch.randn(32, 5760, generator=g))
        m.mlp2_bias.copy_(0.1 * torch.randn(32, 2880, generator=g))
        for blocks, scales in ((m.mlp1_blocks, m.mlp1_scales), (m.mlp2_blocks, m.mlp2_scales)):
            blocks.copy_(torch.randint(0, 256, blocks.shape, generator=d, dtype=torch.uint8, device="cuda"))
            scales.copy_(torch.randint(118, 122, scales.shape, generator=d, dtype=torch.uint8, device="cuda"))
    return m


def gpt_oss_routing(m, x):
    """The norm's rows, the logits, and which tokens' experts a place of bf16 in a logit cannot change; float64 on the CPU."""
    t = x.double()
    t = (t * torch.rsqrt(t.square().mean(-1, keepdim=True) + m.norm.eps) * m.norm.scale.detach().cpu().double()).bfloat16().double()
    logits = (t @ m.gate.weight.detach().cpu().double().t() + m.gate.bias.detach().cpu().double()).bfloat16().double()
    v, e = torch.sort(logits, dim=1, descending=True, stable=True)
    return t, e[:, :4], torch.softmax(v[:, :4], 1), v[:, 3] - v[:, 4] > 0.05


@gpu
@pytest.mark.parametrize("tokens", [1, 8, 40, 300])
def test_mlp_block_of_gpt_oss_sizes(tokens):
    m = gpt_oss_block(1)
    x = torch.randn(tokens, 2880, generator=torch.Generator().manual_seed(tokens)).bfloat16()
    t, chosen, weights, sure = gpt_oss_routing(m, x)
    assert sure.double().mean() > 0.7
    want, t, on = x.double().cuda(), t.cuda(), lambda p: p.detach().double()
    table = FP4.cuda()

    def dense(blocks, scales):
        v = torch.stack((table[(blocks & 15).int()], table[(blocks >> 4).int()]), -1).flatten(-2)
        return (v * torch.exp2(scales.double() - 127)[..., None]).flatten(-2)

    for e in range(32):
        at, j = (chosen == e).cuda().nonzero(as_tuple=True)
        if len(at):
            y = t[at] @ dense(m.mlp1_blocks[e], m.mlp1_scales[e]).t() + on(m.mlp1_bias[e])
            gate, lin = y[:, 0::2].clamp(max=LIMIT), y[:, 1::2].clamp(-LIMIT, LIMIT)
            h = (gate * torch.sigmoid(ALPHA * gate) * (lin + 1)).bfloat16().double()
            want.index_add_(0, at, weights.cuda()[at, j, None] * (h @ dense(m.mlp2_blocks[e], m.mlp2_scales[e]).t() + on(m.mlp2_bias[e])))
    got = m(x.cuda())
    # (as for the small blocks: a place of bf16 in t, the logits and h each, and in the result)
    torch.testing.assert_close(got.double().cpu()[sure], want.cpu()[sure], rtol=2e-2, atol=2e-2)


@gpu
def test_mlp_block_of_one_token():
    """One token whose experts are sure, for each of several."""
    m = mlp_block()
    x = torch.randn(24, 192, generator=torch.Generator().manual_seed(3)).bfloat16()
    want, sure = block_ref(m, x)
    assert sure.sum() > 12
    for i in sure.nonzero()[:, 0].tolist():
        torch.testing.assert_close(m(x[i: i + 1].cuda()).double().cpu(), want[i: i + 1], rtol=2e-2, atol=2e-2)


@gpu
@pytest.mark.parametrize("tokens", [6, 130])
@pytest.mark.parametrize("experts,top", [(17, 3), (5, 4)])
def test_mlp_block_of_an_odd_number_of_experts(tokens, experts, top):
    m = mlp_block(experts=experts, top=top)
    x = torch.randn(tokens, 192, generator=torch.Generator().manual_seed(tokens)).bfloat16()
    want, sure = block_ref(m, x)
    assert sure.double().mean() > 0.5
    torch.testing.assert_close(m(x.cuda()).double().cpu()[sure], want[sure], rtol=2e-2, atol=2e-2)


@gpu
def test_mlp_block_in_a_graph():
    """Nothing of a call lives on the host: a captured block replays with other tokens, also other experts, and between eager work."""
    m = mlp_block()
    for tokens in (3, 100):
        x = torch.randn(tokens, 192, device="cuda").bfloat16()
        m(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m(x)
        for seed in range(4):
            x.copy_(torch.randn(tokens, 192, generator=torch.Generator().manual_seed(seed)))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, m(x))


@gpu
def test_ops_on_two_streams():
    """Outputs and workspaces belong to a call: the same calls on two streams at once give what they give alone."""
    m = mlp_block()
    xs = [torch.randn(200, 192, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i in range(2)]
    want = [m(x) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                t = T.router_logits(xs[i], m.gate.weight.detach(), m.gate.bias.detach())          # (the norm's buffer is borrowed: one stream's at a time)
                r = T.moe_route(t, 4)
                h = T.moe_mlp1(xs[i], r, m.mlp1_blocks, m.mlp1_scales, m.mlp1_bias.detach())
                got[i].append(T.moe_mlp2(h, r, m.mlp2_blocks, m.mlp2_scales, m.mlp2_bias.detach(), residual=xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        r = T.moe_route(T.router_logits(xs[i], m.gate.weight.detach(), m.gate.bias.detach()), 4)
        h = T.moe_mlp1(xs[i], r, m.mlp1_blocks, m.mlp1_scales, m.mlp1_bias.detach())
        alone = T.moe_mlp2(h, r, m.mlp2_blocks, m.mlp2_scales, m.mlp2_bias.detach(), residual=xs[i])
        assert all(torch.equal(g, alone) for g in got[i]) and want[i].shape == alone.shape


@gpu
@pytest.mark.parametrize("tokens", [2, 70])
def test_mlp_block_of_a_borrowed_buffer(tokens):
    """The rows that a norm has lent out are rows as others: the block's own norm leaves them alone, and the residual is theirs."""
    m, before = mlp_block(), T.RMSNorm(192, device="cuda")
    rows = torch.randn(tokens, 192, generator=torch.Generator().manual_seed(tokens)).bfloat16().cuda()
    for shape in ((tokens, 192), (1, tokens, 192)):
        x = before(rows.view(shape))                               # (the pool's buffer of this shape)
        kept = x.clone()
        want = m(kept)
        assert torch.equal(m(x), want) and torch.equal(x, kept)
    wide = torch.cat([rows, rows], 1)[:, 3:195]                    # rows that lie apart
    assert torch.equal(m(wide), m(wide.contiguous()))


@gpu
def test_mlp_blocks_on_two_streams():
    """Two blocks of one shape, each on its stream at the same time, give what they give alone."""
    ms = [mlp_block(seed=i) for i in range(2)]
    xs = [torch.randn(200, 192, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i in range(2)]
    want = [m(x) for m, x in zip(ms, xs)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in ms], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ms[i](xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@gpu
def test_mlp_block_from_a_checkpoint(tmp_path):
    from safetensors.torch import save_file

    m = mlp_block(seed=3)
    n = "block.1.mlp."
    save_file({n + "norm.scale": m.norm.scale.detach().cpu().clone(), n + "gate.weight": m.gate.weight.detach().cpu().clone(),
               n + "gate.bias": m.gate.bias.detach().cpu().clone(), n + "mlp1_bias": m.mlp1_bias.detach().cpu().clone(),
               n + "mlp2_bias": m.mlp2_bias.detach().cpu().clone(), n + "mlp1_weight.blocks": m.mlp1_blocks.cpu(), n + "mlp1_weight.scales": m.mlp1_scales.cpu(),
               n + "mlp2_weight.blocks": m.mlp2_blocks.cpu(), n + "mlp2_weight.scales": m.mlp2_scales.cpu()}, str(tmp_path / "a.safetensors"))
    ck = T.Checkpoint(str(tmp_path), torch.device("cuda"))
    with pytest.raises(AssertionError, match="not stored in MXFP4"):
        ck.get_mxfp4(n + "mlp1_bias")
    loaded = T.MLPBlock(192, 160, 16, 4, device="cuda").load(ck, 1)
    x = torch.randn(11, 192, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    assert torch.equal(loaded(x), m(x))
    expanded = ck.get(n + "mlp1_weight")                           # the same weights, expanded: what the products multiply with
    assert torch.equal(expanded.double().cpu(), values(m.mlp1_blocks.cpu(), m.mlp1_scales.cpu()))


# ---- refusals ---------------------------------------------------------------------------------------------------------------
def _err():
    return _lib.lib().tllm_last_error().decode()


def test_entry_points_refuse_what_they_cannot_do():
    lib, p, odd = _lib.lib(), C.c_void_p(4096), C.c_void_p(4104)
    q = lib.tllm_mxfp4_quantize
    assert q(None, 0, 0, None, None, 0, 64, None) == 0 and q(None, 0, 0, None, None, 3, 0, None) == 0
    assert q(p, 0, 64, p, p, -1, 64, None) == -1 and q(p, 3, 64, p, p, 1, 64, None) == -1 and "type" in _err()
    assert q(p, 0, 40, p, p, 2, 40, None) == -2 and q(None, 0, 64, p, p, 2, 64, None) == -1
    assert q(p, 0, 32, p, p, 2, 64, None) == -1 and q(odd, 0, 64, p, p, 2, 64, None) == -3 and q(p, 0, 66, p, p, 2, 64, None) == -3
    lin = lib.tllm_mxfp4_linear_bf16
    assert lin(None, None, 0, None, None, None, None, 0, 0, 64, 64, None) == 0
    assert lin(p, None, 64, p, p, None, p, 16, -1, 64, 16, None) == -1
    assert lin(p, None, 48, p, p, None, p, 16, 2, 48, 16, None) == -2 and "32" in _err()
    assert lin(p, None, 64, p, p, None, p, 16, 2, 64, 0, None) == -2
    assert lin(p, None, 32, p, p, None, p, 16, 2, 64, 16, None) == -1 and lin(p, None, 64, p, p, None, p, 8, 2, 64, 16, None) == -1
    assert lin(odd, None, 64, p, p, None, p, 16, 2, 64, 16, None) == -3 and lin(p, None, 64, odd, p, None, p, 16, 2, 64, 16, None) == -3
    assert lin(p, None, 68, p, p, None, p, 16, 2, 64, 16, None) == -3
    assert lin(p, None, 64, None, p, None, p, 16, 2, 64, 16, None) == -1 and lin(p, None, 64, p, p, None, None, 16, 2, 64, 16, None) == -1
    assert lin(p, None, 1 << 25, p, p, None, p, 16, 300, 4096, 16, None) == -2 and "4 GiB" in _err()
    r = lib.tllm_moe_route

    def route(logits=p, stride=32, groups=1, kept=1, tokens=8, experts=32, top=4, work=None, nbytes=0, offsets=p):
        return r(logits, 0, stride, None, 0, groups, kept, 1, 1.0, p, p, p, offsets, work, nbytes, tokens, experts, top, None)

    assert route(tokens=-1) == -1 and route(experts=0) == -2 and route(experts=513, stride=513) == -2 and route(top=0) == -2 and route(top=33) == -2
    assert route(groups=5) == -2 and route(groups=4, kept=5) == -2 and route(groups=4, kept=0) == -2 and route(groups=16, kept=1) == -2
    assert route(stride=31) == -1 and route(logits=None) == -1 and route(offsets=None) == -1 and route(tokens=1 << 30) == -2
    need = lib.tllm_moe_route_workspace_bytes(1000, 32)
    assert need > 0 and lib.tllm_moe_route_workspace_bytes(8, 32) == 0
    assert route(tokens=1000) == -1 and route(tokens=1000, work=p, nbytes=need - 1) == -1 and "workspace" in _err()

    def mlp1(x=p, stride=64, order=p, w=p, h=p, h_stride=32, tokens=8, experts=4, top=2, hidden=64, inner=32, limit=7.0):
        return lib.tllm_moe_mlp1_bf16(x, stride, order, p, w, p, None, h, h_stride, tokens, experts, top, hidden, inner, 1.702, limit, 1, None)

    assert mlp1(tokens=0) == 0 and mlp1(tokens=-1) == -1 and mlp1(top=0) == -2 and mlp1(top=5) == -2 and mlp1(hidden=40, stride=40) == -2
    assert mlp1(x=None) == -1 and mlp1(order=None) == -1 and mlp1(w=odd) == -3 and mlp1(x=odd) == -3 and mlp1(h=None) == -1 and mlp1(h_stride=31) == -1
    assert mlp1(tokens=1 << 20, stride=4096) == -2 and "4 GiB" in _err()
    assert mlp1(stride=32) == -1 and mlp1(limit=-1.0) == -1 and mlp1(tokens=1 << 30) == -2 and mlp1(inner=0) == -2

    def mlp2(h=p, weights=p, out=p, out_stride=64, work=p, nbytes=8 * 2 * 64 * 4, tokens=8, experts=4, top=2, inner=32, hidden=64, res=None, res_stride=64):
        return lib.tllm_moe_mlp2_bf16(h, inner, p, p, weights, p, p, None, res, res_stride, out, out_stride, work, nbytes, tokens, experts, top, inner, hidden, None)

    assert lib.tllm_moe_mlp2_workspace_bytes(8, 2, 64) <= 8 * 2 * 64 * 4
    assert mlp2(tokens=0) == 0 and mlp2(tokens=-1) == -1 and mlp2(h=None) == -1 and mlp2(weights=None) == -1 and mlp2(out=None) == -1
    assert mlp2(out_stride=63) == -1 and mlp2(res=p, res_stride=63) == -1 and mlp2(inner=33) == -2
    assert lib.tllm_moe_mlp2_workspace_bytes(300, 2, 64) > 16 and mlp2(tokens=300, nbytes=16) == -1 and "workspace" in _err()


def test_rows_beyond_the_longest_are_refused():
    lib, p = _lib.lib(), C.c_void_p(4096)
    k = (1 << 18) + 32
    assert lib.tllm_mxfp4_linear_bf16(p, None, k, p, p, None, p, 16, 2, k, 16, None) == -2 and "too large" in _err()
    assert lib.tllm_mxfp4_linear_bf16(p, p, 0, p, p, None, p, 16, 2, k, 16, None) == -2 and "too large" in _err()
    assert lib.tllm_moe_mlp1_bf16(p, k, p, p, p, p, None, p, 32, 8, 4, 2, k, 32, 1.702, 7.0, 1, None) == -2 and "too large" in _err()


def test_ops_refuse_cpu_tensors():
    x, u8 = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 16, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="GPU only"):
        T.mxfp4_quantize(x)
    with pytest.raises(RuntimeError, match="GPU only"):
        T.mxfp4_linear(x, u8, u8[..., 0])
    with pytest.raises(RuntimeError, match="GPU only"):
        T.moe_route(x, 2)
    routing = T.MoeRouting(torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, 1), torch.arange(2, dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32))
    for op in (T.moe_mlp1, T.moe_mlp2):
        with pytest.raises(RuntimeError, match="GPU only"):
            op(x, routing, u8[None], u8[None, ..., 0])


def test_linear_operands_with_a_bias_of_another_length_are_refused():
    """The kernels read a bias value for each row of the weight: one that is shorter would be read beyond its end."""
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(32, 64, dtype=torch.bfloat16)
    for n in (0, 1, 31, 33):
        with pytest.raises(AssertionError, match=f"{n} values for 32"):
            T.ops._prep_linear(x, w, torch.zeros(n, dtype=torch.bfloat16))
    T.ops._prep_linear(x, w, torch.zeros(32, dtype=torch.bfloat16))
    T.ops._prep_linear(x, w, None)


@gpu
@pytest.mark.parametrize("tokens", [1, 65])
@pytest.mark.parametrize("experts", [32, 10])
def test_router_logits_refuses_a_bias_of_another_length(tokens, experts):
    x, w = torch.zeros(tokens, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(experts, 64, dtype=torch.bfloat16, device="cuda")
    for n in (1, experts - 1, experts + 1):
        for op in (T.router_logits, T.linear_qkv_forward):
            with pytest.raises(AssertionError, match="bias"):
                op(x, w, torch.zeros(n, dtype=torch.bfloat16, device="cuda"))


@gpu
def test_products_over_rows_of_no_values_are_refused():
    """K = 0, with both types of activations; without rows or without outputs there is nothing to compute."""
    u8 = lambda *shape: torch.zeros(shape, dtype=torch.uint8, device="cuda")
    bf = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
    for lead in ((3,), (2, 5), ()):
        for bias in (None, bf(6)):
            with pytest.raises(RuntimeError, match="whole blocks"):
                T.mxfp4_linear(u8(*lead, 0, 16), u8(6, 0, 16), u8(6, 0), bias, x_scales=u8(*lead, 0))
    with pytest.raises(RuntimeError, match="whole blocks"):
        T.mxfp4_linear(bf(3, 0), u8(6, 0, 16), u8(6, 0))
    assert T.mxfp4_linear(u8(0, 2, 16), u8(6, 2, 16), u8(6, 2), x_scales=u8(0, 2)).shape == (0, 6)
    assert T.mxfp4_linear(u8(4, 2, 16), u8(0, 2, 16), u8(0, 2), x_scales=u8(4, 2)).shape == (4, 0)
    routing = T.moe_route(torch.zeros(2, 3, device="cuda"), 1)
    for op in (T.moe_mlp1, T.moe_mlp2):
        with pytest.raises(RuntimeError, match="whole blocks"):
            op(bf(2, 0), routing, u8(3, 4, 0, 16), u8(3, 4, 0))


@gpu
def test_ops_refuse_wrong_types_and_shapes():
    c = dict(device="cuda")
    x, w, ws = torch.zeros(2, 64, dtype=torch.bfloat16, **c), torch.zeros(6, 2, 16, dtype=torch.uint8, **c), torch.zeros(6, 2, dtype=torch.uint8, **c)
    good = T.moe_route(torch.zeros(2, 3, **c), 1)
    w3, ws3 = w.view(3, 2, 2, 16), ws.view(3, 2, 2)
    bad = [lambda: T.mxfp4_quantize(x.double()), lambda: T.mxfp4_quantize(x[:, :40]), lambda: T.mxfp4_linear(x.float(), w, ws),
           lambda: T.mxfp4_linear(x[:, :32], w, ws), lambda: T.mxfp4_linear(x, w, ws[:, :1]), lambda: T.mxfp4_linear(x, w[..., :8], ws),
           lambda: T.mxfp4_linear(x, w.int(), ws), lambda: T.mxfp4_linear(x, w, ws, torch.zeros(5, dtype=torch.bfloat16, **c)),
           lambda: T.mxfp4_linear(x, w, ws, torch.zeros(6, **c)), lambda: T.mxfp4_linear(w, w, ws, x_scales=ws[:, :1]),
           lambda: T.mxfp4_linear(x, w, ws, x_scales=ws), lambda: T.moe_route(x.half(), 2), lambda: T.moe_route(x, 2, score="tanh"),
           lambda: T.moe_route(x, 2, bias=torch.zeros(63, **c)), lambda: T.moe_route(x, 2, bias=torch.zeros(64, dtype=torch.bfloat16, **c)),
           lambda: T.moe_mlp1(x[:1], good, w3, ws3), lambda: T.moe_mlp1(x[:, :32], good, w3, ws3), lambda: T.moe_mlp1(x, good, w3[:2], ws3[:2]),
           lambda: T.moe_mlp1(x, good._replace(order=good.order.long()), w3, ws3), lambda: T.moe_mlp1(x, good, w3[:, :1], ws3[:, :1]),
           lambda: T.moe_mlp2(x[:1], good, w3, ws3), lambda: T.moe_mlp2(x, good, w3, ws3, residual=x),
           lambda: T.moe_mlp2(x, good, w3, ws3, out=torch.zeros(2, 3, dtype=torch.bfloat16, **c))]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            print("call", i, "was let through")
    with pytest.raises(RuntimeError, match="top"):
        T.moe_route(x, 65)
