"""8-bit float quantisation and products with block scales (bm_fp8_quantize,
bm_fp8_product, bm_fp8_logits) against their definitions in 64 bits."""
import ctypes

import numpy as np
import pytest

DEFAULT = 1
U = 2.0 ** -24


def pitch(rows):
    return -(-rows // 4) * 4


def quantize(gpu_ctx, x, w=None, ldx=None, lds=None):
    import torch
    rows, d = x.shape
    lds = lds or pitch(rows)
    q = torch.full((rows, d), 99, dtype=torch.uint8, device="cuda")
    scale = torch.full((-(-d // 128), lds), -5.0, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.fp8_quantize(x.data_ptr(), "f32" if x.dtype == torch.float32 else "bf16", rows, d, ldx or x.stride(0),
                         None if w is None else w.data_ptr(), q.data_ptr(), scale.data_ptr(), lds, DEFAULT)
    torch.cuda.synchronize()
    return q.view(torch.float8_e4m3fn), scale


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("rows,d", [(1, 16), (1, 128), (3, 144), (9, 512), (5, 528), (2, 2048), (33, 2064), (4, 4096),
                                    (2, 4112), (3, 16384)])
def test_quantize(gpu_ctx, type_, norm, rows, d):
    """q is x / scale rounded to e4m3: half a step of the value (2^-4
    relative, 2^-10 below the normal range), plus the roundings of the norm
    (the mean's sum d u, then 6 u) and of the two divisions (2 u); scale is
    max / 448 to the same roundings."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(d)
    t = torch.float32 if type_ == "f32" else torch.bfloat16
    x = (torch.randn(rows, d + 8, generator=g, device="cuda") * torch.exp(torch.randn(rows, d + 8, generator=g, device="cuda"))).to(t)
    x[0, : min(d, 128)] = 0.0
    w = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")) if norm else None
    q, scale = quantize(gpu_ctx, x[:, :d], w, ldx=d + 8, lds=pitch(rows) + 4)
    v = x[:, :d].double().cpu().numpy()
    eps = 2 * U
    if norm:
        v = v / np.sqrt((v * v).mean(1, keepdims=True) + 1e-6) * w.double().cpu().numpy()
        eps += (d + 6) * U
    KB = scale.shape[0]
    for k in range(KB):
        part = v[:, 128 * k:128 * (k + 1)]
        top = np.abs(part).max(1)
        want = np.where(top > 2.0 ** -100, top / 448.0, 1.0)
        s = scale[k, :rows].double().cpu().numpy()
        assert (np.abs(s - want) <= eps * want * 1.01).all()
        got = q[:, 128 * k:128 * (k + 1)].double().cpu().numpy()
        e = part / s[:, None]
        step = np.maximum(2.0 ** -4 * np.abs(e), 2.0 ** -10)
        assert (np.abs(got - e) <= step + 2 * eps * np.abs(e)).all()
    assert (scale[:, rows:] == -5.0).all()  # behind the last row nothing is written


@pytest.mark.gpu
def test_quantize_rounds_to_even_exactly(gpu_ctx):
    """With a block's largest value 448 the scale is 1: every half-way value
    and every e4m3 value."""
    import torch
    v = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    half = (v[:-1] + v[1:]) / 2
    x = torch.cat([v, half, -v, -half])
    x = torch.nn.functional.pad(x, (0, -x.numel() % 127)).view(-1, 127)
    x = torch.cat([x, torch.full((x.shape[0], 1), 448.0)], 1)
    q, scale = quantize(gpu_ctx, x.cuda())
    assert (scale[:, :x.shape[0]] == 1.0).all()
    assert torch.equal(q.cpu().float(), x.to(torch.float8_e4m3fn).float())


@pytest.mark.gpu
def test_quantize_every_bf16_value(gpu_ctx):
    """All pairs of a bf16 significand with a largest of its block, over the
    exponents where e4m3 has values: ties among them."""
    import torch
    sig = (128 + torch.arange(128, device="cuda")).float()
    blocks = []
    for e in range(-2, 20):
        for top in range(128):
            b = sig * 2.0 ** -e
            m = (128.0 + top) * 4
            blocks.append(torch.cat([b[:64], -b[64:127], torch.tensor([m], device="cuda")]).clamp(-m, m))
    x = torch.stack(blocks).to(torch.bfloat16)
    q, _ = quantize(gpu_ctx, x)
    v = x.double()
    v = 448.0 * v / v.abs().amax(1, keepdim=True)
    grid = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    t = v / grid  # (a quotient of 64 bits is exact on a tie, and far from one elsewhere)
    assert torch.equal(q.double(), torch.round(t) * grid)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_quantize_rounds_the_weighted_values_exactly(gpu_ctx, type_):
    """With a norm too, q is what 64 bits give for x * weight / max, value by
    value: the norm's factor drops out.  (A quotient of 64 bits closer than
    2^-46 steps to a border is left out; there are none expected.)"""
    import torch
    rows, d = 1024, 2048
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(rows, d, generator=g, device="cuda").to(torch.float32 if type_ == "f32" else torch.bfloat16)
    w = 1 + 0.02 * torch.randn(d, generator=g, device="cuda")
    q, _ = quantize(gpu_ctx, x, w)
    v = (x.double() * w.double()).view(rows, -1, 128)
    v = (448.0 * v / v.abs().amax(2, keepdim=True)).view(rows, d)
    grid = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    t = v / grid
    sure = ((t - torch.floor(t) - 0.5).abs() > 2.0 ** -46) | (t == torch.round(t))
    assert torch.equal(q.double()[sure], (torch.round(t) * grid)[sure])
    assert sure.float().mean() > 0.9999


@pytest.mark.gpu
def test_quantize_special_values(gpu_ctx):
    import torch
    x = torch.randn(6, 256, device="cuda")
    x[0, 3] = float("nan")
    x[1, 200] = float("inf")
    x[2] = 0.0
    x[3] = 1e-35
    x[4, :128] = 3e38
    q, s = quantize(gpu_ctx, x)
    f = q.float()
    assert s[0, 0].isnan() and f[0, :128].isnan().all() and not f[0, 128:].isnan().any()
    assert s[1, 1].isinf() and f[1, 200].isnan() and (f[1, 128:200] == 0).all()
    assert (s[:, 2:4] == 1.0).all() and (f[2:4] == 0).all()
    assert (f[4, :128] == 448).all()


def product_ref(a, asc, w, wsc):
    M, K = a.shape
    N = w.shape[0]
    out, mag = np.zeros((M, N)), np.zeros((M, N))
    for k in range(-(-K // 128)):
        c = slice(128 * k, min(K, 128 * k + 128))
        s = asc[k, :M, None] * np.repeat(wsc[:, k], 128)[None, :N]
        out += (a[:, c] @ w[:, c].T) * s
        mag += (np.abs(a[:, c]) @ np.abs(w[:, c]).T) * s
    return out, mag


def make(seed, M, K, N):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    f8 = torch.float8_e4m3fn
    a = (torch.randn(M, K, generator=g, device="cuda") * 60).clamp(-448, 448).to(f8)
    w = (torch.randn(N, K, generator=g, device="cuda") * 60).clamp(-448, 448).to(f8)
    KB, NB = -(-K // 128), -(-N // 128)
    asc = torch.full((KB, pitch(M)), float("nan"), device="cuda")
    asc[:, :M] = torch.rand(KB, M, generator=g, device="cuda") + 0.1
    wsc = torch.rand(NB, KB, generator=g, device="cuda") + 0.1
    return a, asc, w, wsc


def product(gpu_ctx, a, asc, w, wsc, pad=0, stream=DEFAULT):
    import torch
    M, K = a.shape
    N = w.shape[0]
    out = torch.full((M, N + pad), -3.0, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.fp8_product(a.data_ptr(), asc.data_ptr(), asc.shape[1], M, K, w.data_ptr(), wsc.data_ptr(), N,
                        out.data_ptr(), N + pad, stream)
    torch.cuda.synchronize()
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 15, 17, 33, 64, 65, 100, 129, 256, 300])
@pytest.mark.parametrize("K,N", [(16, 1), (128, 128), (144, 129), (1040, 1000), (2048, 515)])
def test_product(gpu_ctx, M, K, N):
    """The sum of a block of at most 128 products by the tensor core is off by
    at most 128 roundings or truncations of its sum of magnitudes (2 u each),
    the scale product and the scaled blocks' additions by one u each."""
    a, asc, w, wsc = make(M * 7 + K, M, K, N)
    out = product(gpu_ctx, a, asc, w, wsc, pad=M % 3)
    f = lambda t: t.double().cpu().numpy()  # noqa: E731
    want, mag = product_ref(f(a.float()), f(asc), f(w.float()), f(wsc))
    got = f(out)
    assert (np.abs(got[:, :N] - want) <= (256 + 2 + -(-K // 128)) * U * mag).all()
    assert (got[:, N:] == -3.0).all()
    gpu_ctx.check()


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(40, 16384, 300), (700, 512, 20000), (1, 4096, 40001), (513, 128, 385)])
def test_product_many_tiles(gpu_ctx, M, K, N):
    import torch
    a, asc, w, wsc = make(M, M, K, N)
    out = product(gpu_ctx, a, asc, w, wsc)
    ad = a.double() * asc[:, :M].T.double().repeat_interleave(128, 1)[:, :K]
    wd = w.double() * wsc.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    want, mag = ad @ wd.T, ad.abs() @ wd.abs().T
    assert ((out - want).abs() <= (256 + 2 + -(-K // 128)) * U * mag).all()
    gpu_ctx.check()
    assert torch.equal(out, product(gpu_ctx, a, asc, w, wsc))  # the same sums every time


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 31, 48, 66, 95, 96, 97, 128])
@pytest.mark.parametrize("K,N", [(1024, 300), (2000, 9000), (4096, 2047), (4112, 130)])
def test_product_split_over_a_cluster(gpu_ctx, M, K, N):
    """One, two and four CTAs a tile, each with a part of K and of the columns."""
    a, asc, w, wsc = make(K + M, M, K, N)
    out = product(gpu_ctx, a, asc, w, wsc, pad=3)
    ad = a.double() * asc[:, :M].T.double().repeat_interleave(128, 1)[:, :K]
    wd = w.double() * wsc.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    want, mag = ad @ wd.T, ad.abs() @ wd.abs().T
    assert ((out[:, :N] - want).abs() <= (256 + 2 + -(-K // 128)) * U * mag).all()
    assert (out[:, N:] == -3.0).all()
    gpu_ctx.check()


@pytest.mark.gpu
def test_product_nan_stays_in_its_row_and_column(gpu_ctx):
    a, asc, w, wsc = make(3, 20, 256, 300)
    clean = product(gpu_ctx, a, asc, w, wsc)
    a.view(dtype=__import__("torch").uint8)[4, 17] = 0x7F
    w.view(dtype=__import__("torch").uint8)[200, 130] = 0x7F
    got = product(gpu_ctx, a, asc, w, wsc)
    nan = got.isnan()
    assert nan[4].all() and nan[:, 200].all()
    nan[4] = True
    nan[:, 200] = True
    assert ((got == clean) | nan).all() and int(nan.sum()) == 300 + 19


@pytest.mark.gpu
def test_logits_is_quantize_then_product(gpu_ctx):
    import torch
    B, d, V = 37, 2048, 1003
    x = torch.randn(B, d, device="cuda")
    nw = 1 + 0.02 * torch.randn(d, device="cuda")
    _, _, w, wsc = make(5, 1, d, V)
    out = torch.full((B, V + 1), -3.0, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    gpu_ctx.fp8_logits(x.data_ptr(), B, d, nw.data_ptr(), w.data_ptr(), wsc.data_ptr(), V, out.data_ptr(), V + 1,
                       s.cuda_stream)
    torch.cuda.synchronize()
    q, sc = quantize(gpu_ctx, x, nw)
    assert torch.equal(out[:, :V], product(gpu_ctx, q, sc, w, wsc))
    assert (out[:, V] == -3.0).all()
    # captured, replayed on another input
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        gpu_ctx.fp8_logits(x.data_ptr(), B, d, nw.data_ptr(), w.data_ptr(), wsc.data_ptr(), V, out.data_ptr(), V + 1,
                           torch.cuda.current_stream().cuda_stream)
    x.normal_()
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    q, sc = quantize(gpu_ctx, x, nw)
    assert torch.equal(out[:, :V], product(gpu_ctx, q, sc, w, wsc))


def test_refusals(sampler_lib):
    L = sampler_lib.lib()
    ctx = ctypes.create_string_buffer(1 << 16)
    q = 1 << 20
    quant = dict(ctx=ctx, x=q, type=0, rows=5, d=256, ldx=256, w=q, q=q, s=q, lds=8, stream=None)
    prod = dict(ctx=ctx, a=q, asc=q, lds=8, rows=5, d=256, w=q, wsc=q, n=100, out=q, ldo=100, stream=None)
    logits = dict(ctx=ctx, x=q, B=5, d=256, nw=q, w=q, wsc=q, V=100, out=q, ld=100, stream=None)

    def refuses(f, base, **ch):
        a = dict(base)
        a.update(ch)
        return f(*a.values()) in (-1, -4)

    for ch in (dict(ctx=None), dict(x=None), dict(x=q + 8), dict(type=2), dict(rows=-1), dict(d=0), dict(d=8), dict(d=24),
               dict(d=16400), dict(ldx=252), dict(ldx=258), dict(w=q + 4), dict(q=None), dict(q=q + 4), dict(s=None),
               dict(s=q + 4), dict(lds=4), dict(lds=6)):
        assert refuses(L.bm_fp8_quantize, quant, **ch), ch
    for ch in (dict(ctx=None), dict(a=None), dict(a=q + 8), dict(asc=None), dict(asc=q + 4), dict(lds=4), dict(lds=6),
               dict(rows=-1), dict(d=24), dict(d=16400), dict(w=None), dict(w=q + 8), dict(wsc=None), dict(wsc=q + 2),
               dict(n=0), dict(out=None), dict(out=q + 2), dict(ldo=99)):
        assert refuses(L.bm_fp8_product, prod, **ch), ch
    for ch in (dict(ctx=None), dict(x=None), dict(x=q + 4), dict(B=-1), dict(d=24), dict(nw=q + 4), dict(V=0), dict(ld=99)):
        assert refuses(L.bm_fp8_logits, logits, **ch), ch
    for f, base, k in ((L.bm_fp8_quantize, quant, "rows"), (L.bm_fp8_product, prod, "rows"), (L.bm_fp8_logits, logits, "B")):
        assert f(*{**base, k: 0}.values()) == 0


def test_refuses_rows_whose_tiles_overflow(sampler_lib):
    L = sampler_lib.lib()
    ctx = ctypes.create_string_buffer(1 << 16)
    q, most = 1 << 20, 2 ** 31 - 1
    assert L.bm_fp8_quantize(ctx, q, 0, most, 16, 16, q, q, q, most + 1, None) == -4
    assert L.bm_fp8_product(ctx, q, q, most + 1, most, 16, q, q, 100, q, 100, None) == -4
    assert L.bm_fp8_product(ctx, q, q, 8, 5, 16, q, q, most, q, most, None) == -4
    assert L.bm_fp8_logits(ctx, q, most, 16, q, q, q, 100, q, 100, None) == -4


@pytest.mark.gpu
def test_products_at_once_on_two_streams(gpu_ctx):
    """One context, no workspace: calls of both kinds of tile may overlap."""
    import torch
    few, many = make(21, 20, 2048, 4000), make(22, 700, 1024, 3000)
    want = product(gpu_ctx, *few), product(gpu_ctx, *many)
    outs = [torch.full_like(w, -3.0) for w in want]
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(4):
        for (a, asc, w, wsc), out, s in zip((few, many), outs, streams):
            gpu_ctx.fp8_product(a.data_ptr(), asc.data_ptr(), asc.shape[1], a.shape[0], a.shape[1], w.data_ptr(),
                                wsc.data_ptr(), w.shape[0], out.data_ptr(), w.shape[0], s.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    gpu_ctx.check()


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(97, 8192, 10000), (128, 8192, 10000), (128, 14976, 9600), (100, 16384, 9600),
                                   (128, 16384, 9000), (97, 13584, 4800), (200, 16384, 3200)])
def test_product_with_few_stages(gpu_ctx, M, K, N):
    """Tiles of 128 rows whose scales leave room for four stages, whole rows of
    K and parts of it: bounds as for test_product, twice with the same sums."""
    import torch
    a, asc, w, wsc = make(M + K, M, K, N)
    out = product(gpu_ctx, a, asc, w, wsc)
    ad = a.double() * asc[:, :M].T.double().repeat_interleave(128, 1)[:, :K]
    wd = w.double() * wsc.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    want, mag = ad @ wd.T, ad.abs() @ wd.abs().T
    assert ((out - want).abs() <= (256 + 2 + -(-K // 128)) * U * mag).all()
    assert torch.equal(out, product(gpu_ctx, a, asc, w, wsc))
    gpu_ctx.check()


def codes_of(v):
    """e4m3 values of 448 v / max|v| by blocks of 128 columns, from 64 bits, and
    where a quotient is too close to a border to tell (closer than 2^-46 steps)."""
    import torch
    b = v.view(v.shape[0], -1, 128)
    b = (448.0 * b / b.abs().amax(2, keepdim=True)).view(v.shape)
    grid = torch.exp2(torch.floor(torch.log2(b.abs().clamp(min=2.0 ** -6))) - 3)
    t = b / grid
    sure = ((t - torch.floor(t) - 0.5).abs() > 2.0 ** -46) | (t == torch.round(t))
    return torch.round(t) * grid, sure


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_quantize_at_the_ends_of_the_range(gpu_ctx, type_):
    """Finite blocks whose largest lies in [2^115, 2^128) or [2^-100, 2^-97):
    finite scales (a division's rounding off) and the codes of the exact
    quotients.  In bf16 every significand of a value and of the largest, ties
    among them: there a quotient is on a border or 2^-16 away."""
    import torch
    t = torch.float32 if type_ == "f32" else torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(6)
    bits = 24 if type_ == "f32" else 8
    blocks = []
    for e in list(range(115, 128)) + [-99, -98, -97]:
        n = 128
        top = 1.0 + torch.arange(n, device="cuda").double() / n
        sig = 2 ** (bits - 1) + torch.randint(0, 2 ** (bits - 1), (n, 128), generator=g, device="cuda")
        if type_ == "bf16":
            sig = (128 + torch.arange(128, device="cuda")).expand(n, 128)
        v = sig.double() / 2 ** (bits - 1) * torch.exp2(-torch.randint(0, 18, (n, 128), generator=g, device="cuda").double())
        v = v * torch.where(torch.rand(n, 128, generator=g, device="cuda") < 0.5, -1.0, 1.0)
        v = torch.maximum(torch.minimum(v, top[:, None]), -top[:, None])
        v[:, 5] = top
        blocks.append(v * 2.0 ** e)
    x = torch.cat(blocks).to(t)
    assert torch.equal(x.double(), torch.cat(blocks))
    q, scale = quantize(gpu_ctx, x)
    want, sure = codes_of(x.double())
    if type_ == "bf16":  # a quotient of 64 bits is exact on a tie, and far from one elsewhere
        sure |= True
    assert torch.equal(q.double()[sure], want[sure]) and sure.float().mean() > 0.9999
    exact = x.double().abs().amax(1) / 448.0
    assert ((scale[0, :x.shape[0]].double() - exact).abs() <= 2 * U * exact).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("ex,ew", [(0, 118), (0, 126), (3, 127), (-30, 127), (-52, -52), (-55, -50), (0, -99), (50, 80)])
def test_quantize_with_a_norm_at_the_ends(gpu_ctx, type_, ex, ew):
    """x about 2^ex, weights about 2^ew: products near the ends of the range and
    past it; the scale is max|x w| / rms / 448 to the roundings of
    test_quantize."""
    import torch
    rows, d = 64, 512
    g = torch.Generator(device="cuda").manual_seed(7)
    x = (torch.randn(rows, d, generator=g, device="cuda") * 2.0 ** ex).to(torch.float32 if type_ == "f32" else torch.bfloat16)
    w = (1.0 + 0.9 * torch.rand(d, generator=g, device="cuda")) * 2.0 ** ew
    q, scale = quantize(gpu_ctx, x, w)
    v = x.double() * w.double()
    want, sure = codes_of(v)
    assert torch.equal(q.double()[sure], want[sure]) and sure.float().mean() > 0.9999
    rms = torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + 1e-6)
    exact = (v.abs() / rms).view(rows, -1, 128).amax(2).T / 448.0
    assert ((scale[:, :rows].double() - exact).abs() <= (d + 8) * U * exact * 1.01).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_quantize_special_values_with_a_norm(gpu_ctx, type_):
    """A NaN makes its row's factor NaN, an infinity 0; so do squares past the
    range of fp32, whose row becomes zeros."""
    import torch
    x = torch.randn(5, 384, device="cuda")
    x[0, 3] = float("nan")
    x[1, 200] = -float("inf")
    x[2] *= 2.0 ** 80
    w = 1 + 0.1 * torch.rand(384, device="cuda")
    q, s = quantize(gpu_ctx, x.to(torch.float32 if type_ == "f32" else torch.bfloat16), w)
    f, s = q.float(), s.T
    assert s[0].isnan().all() and f[0].isnan().all()
    assert s[1, 1].isnan() and f[1, 128:256].isnan().all()
    assert (s[1, [0, 2]] == 1.0).all() and (f[1, :128] == 0).all() and (f[1, 256:] == 0).all()
    assert (s[2] == 1.0).all() and (f[2] == 0).all()
    w[5] = float("inf")
    q, s = quantize(gpu_ctx, x.to(torch.float32 if type_ == "f32" else torch.bfloat16), w)
    f, s = q.float(), s.T
    assert s[3:5, 0].isinf().all() and f[3:5, 5].isnan().all() and (f[3:5, 6:128] == 0).all()
    assert s[3:5, 1:].isfinite().all() and f[3:5, 128:].isfinite().all()


def test_logits_refuses_the_products_operands_first(sampler_lib):
    """Before the rows are quantised (the context stands for a real one)."""
    L = sampler_lib.lib()
    ctx = ctypes.create_string_buffer(1 << 16)
    q = 1 << 20
    for w, wsc, out in ((None, q, q), (q + 8, q, q), (q, None, q), (q, q + 2, q), (q, q, None), (q, q, q + 1)):
        assert L.bm_fp8_logits(ctx, q, 5, 256, q, w, wsc, 100, out, 100, None) == -1
