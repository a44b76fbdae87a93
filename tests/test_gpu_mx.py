"""Microscaled blocks on the GPU against their float64 definitions: codes and scale bytes bit for bit where the input
is given, within the roundings of fp32 behind the norm and the activation; the product within those of its sum."""

import math

import numpy as np
import pytest

import mx_helpers as H
from gpu_helpers import log

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FMTS = ["e4m3", "e2m1"]
NORM_REL = 2.0 ** -18  # 64 additions and products of 2^-24 each in a row's sum, halved by the root, and four more
ACT_REL = 2.0 ** -16   # e^-g to |g| log2(e) 2^-24 and some 2^-22, |g| up to 100


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda", 0)


def _spread(rows, cols, seed, dtype=torch.float32, span=3.0):
    """Values whose blocks and members differ widely in size, some on the borders between codes, zeros among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(span * torch.randn(rows, cols, generator=g))
    at = torch.rand(rows, cols, generator=g)
    x = torch.where(at < 0.2, (x * 16).round() / 16, x)
    x = torch.where(at > 0.95, torch.zeros_like(x), x)
    x = torch.where((at > 0.93) & (at < 0.95), -torch.zeros_like(x), x)
    return x.clamp(-6e4, 6e4).to(dtype)


def _random_blocks(rows, cols, fmt, seed, lo=117, hi=131):
    """Any codes but NaN, scales within 2^14 of each other."""
    from pgmoe import MXTensor
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256 if fmt == "e4m3" else 16, (rows, cols), generator=g)
    if fmt == "e4m3":
        codes = torch.where(codes % 128 == 127, torch.zeros_like(codes), codes)
    e = torch.randint(lo, hi, (rows, cols // 32), generator=g)
    t = MXTensor(H.pack(codes, fmt).to("cuda"), e.to(torch.uint8).to("cuda"), fmt)
    return t, H.decode(codes, e, fmt)


# ---------------------------------------------------------------- blocks
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 4096), (3, 96), (7, 1440), (130, 64), (33, 2880), (2050, 512)])
def test_quantize_bits(dev, fmt, dtype, rows, cols):
    from pgmoe import mx_quantize
    x = _spread(rows, cols, rows + cols, dtype)
    t = mx_quantize(x.to(dev), fmt)
    codes, e = H.encode(x, fmt)
    assert t.shape == (rows, cols) and t.fmt == fmt
    assert torch.equal(H.scales(t), e)
    assert torch.equal(H.unpack(t), codes)
    for dt in H.DTYPES:
        v = t.dequantize(dt)
        assert v.dtype == dt and torch.equal(v.cpu(), H.decode(codes, e, fmt).to(dt))


@pytest.mark.parametrize("fmt", FMTS)
def test_every_fp16_value_rounds_as_defined(dev, fmt):
    """All finite fp16 values beside one that fixes the block's power of two, for every power."""
    from pgmoe import mx_quantize
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    every = every[torch.isfinite(every)]
    every = torch.cat((every, every.new_zeros(-len(every) % 31))).reshape(-1, 31)
    for top in (2.0 ** -10, 1.0, 1.75, 448.0, 65504.0):
        x = torch.cat((torch.full((every.shape[0], 1), top, dtype=torch.float16), every.clamp(-top, top)), 1)
        t = mx_quantize(x.to(dev), fmt)
        codes, e = H.encode(x, fmt)
        assert torch.equal(H.scales(t), e) and torch.equal(H.unpack(t), codes)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_far_sizes(dev, fmt):
    """fp32 blocks at the ends of the range: zeros, subnormals, the smallest scale, the largest values."""
    from pgmoe import mx_quantize
    tops = [0.0, 1e-45, 1e-42, 2.0 ** -126, 2.0 ** -120, 2.0 ** -118, 3e-30, 1e30, 2.0 ** 127, 3.4028234e38]
    g = torch.Generator().manual_seed(5)
    x = (2 * torch.rand(len(tops), 32, generator=g) - 1) * torch.tensor(tops)[:, None]
    x[:, 7] = torch.tensor(tops)
    t = mx_quantize(x.to(dev), fmt)
    codes, e = H.encode(x, fmt)
    assert torch.equal(H.scales(t), e) and torch.equal(H.unpack(t), codes)
    assert torch.equal(t.dequantize().cpu(), H.decode(codes, e, fmt).float())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", H.DTYPES)
def test_blocks_that_are_not_finite(dev, fmt, dtype):
    from pgmoe import mx_quantize
    x = _spread(5, 160, 3, dtype)
    x[0, 5], x[1, 64], x[3, 159], x[3, 0] = math.nan, math.inf, -math.inf, math.nan
    t = mx_quantize(x.to(dev), fmt)
    codes, e = H.encode(x, fmt)
    assert torch.equal(H.scales(t), e) and torch.equal(H.unpack(t), codes)
    assert (e == 255).sum() == 4
    v = t.dequantize(torch.float32).cpu()
    assert torch.equal(torch.isnan(v), (e == 255).repeat_interleave(32, 1))


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_takes_views(dev, fmt):
    """Rows apart, transposed, expanded, misaligned, more dimensions, none."""
    from pgmoe import mx_quantize
    base = _spread(64, 512, 9, torch.float16).to(dev)
    views = [base[:, 64:128], base[::3], base[:, 1:97], base.t()[:64, :64], base[:1].expand(5, 512), base[5],
             base.view(4, 16, 512)[:, :3, 32:96], base.view(4, 16, 1, 512), base[:0], base[:1, 40:104]]
    for i, x in enumerate(views):
        t = mx_quantize(x, fmt)
        assert t.shape == tuple(x.shape)
        codes, e = H.encode(x.cpu().reshape(-1, x.shape[-1]), fmt)
        assert torch.equal(H.scales(t), e) and torch.equal(H.unpack(t), codes), i


# ---------------------------------------------------------------- norm and activation
@pytest.mark.parametrize("fmt", FMTS)
def test_vectors_with_gaps(dev, fmt):
    """A single row whose elements do not lie next to each other: of values, codes and scale bytes."""
    from pgmoe import HipMXLinear, MXTensor, exec_fused_act_mul_mx, mx_quantize
    x = _spread(1, 2048, 10).to(dev)[0, ::2]
    t = mx_quantize(x, fmt)
    codes, e = H.encode(x.cpu()[None], fmt)
    assert torch.equal(H.scales(t), e) and torch.equal(H.unpack(t), codes)
    gap = lambda v: torch.stack((v, torch.full_like(v, 3)), 1).flatten()[::2]  # noqa: E731
    again = MXTensor(gap(t.codes), gap(t.scales), fmt)
    assert torch.equal(again.dequantize(), t.dequantize())
    for act in ("silu", "gelu"):
        assert torch.equal(exec_fused_act_mul_mx(x, x, act, fmt).codes, exec_fused_act_mul_mx(x.contiguous(), x.contiguous(), act, fmt).codes)
    layer = HipMXLinear(_random_blocks(40, 1024, "e2m1", 11)[0], act_fmt=fmt)
    assert torch.equal(layer(x), layer(x.contiguous()))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,cols,dt,ddt", [
    (1, 32, torch.float32, None), (1, 4096, torch.float32, torch.float32), (5, 160, torch.float16, torch.bfloat16),
    (9, 288, torch.bfloat16, torch.float32), (3, 1440, torch.float32, torch.float16), (2, 5120, torch.float16, None),
    (70, 64, torch.float32, torch.float32), (2, 8192, torch.bfloat16, torch.bfloat16), (2, 14400, torch.float32, torch.float32),
    (2, 20000, torch.float16, torch.float32), (257, 2048, torch.float32, torch.float32)])
def test_norm(dev, fmt, rows, cols, dt, ddt):
    from pgmoe import exec_fused_add_rmsnorm_mx, exec_fused_rmsnorm_mx
    g = torch.Generator().manual_seed(rows * cols)
    x = (3 * torch.randn(rows, cols, generator=g)).to(dt)
    w = 1 + 0.3 * torch.randn(cols, generator=g)
    h = x.float()
    if ddt is None:
        t = exec_fused_rmsnorm_mx(x.to(dev), w.to(dev), 1e-5, fmt)
    else:
        d = torch.randn(rows, cols, generator=g).to(ddt)
        h = h + d.float()
        got, t = exec_fused_add_rmsnorm_mx(x.to(dev), d.to(dev), w.to(dev), 1e-5, fmt)
        assert got.dtype == torch.float32 and torch.equal(got.cpu(), h)
    h = h.double()
    H.check_blocks(t, h / (h.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double(), NORM_REL)


@pytest.mark.parametrize("rows,cols", [(769, 4096), (900, 2080), (768, 4096)])
def test_norm_of_many_rows(dev, rows, cols):
    """Both divisions of a row among threads, beside each other's sizes."""
    from pgmoe import exec_fused_add_rmsnorm_mx
    x, d = _spread(rows, cols, 16, torch.bfloat16, 1.0), _spread(rows, cols, 17, torch.float32, 1.0)
    w = torch.randn(cols, generator=torch.Generator().manual_seed(18))
    h, t = exec_fused_add_rmsnorm_mx(x.to(dev), d.to(dev), w.to(dev))
    assert torch.equal(h.cpu(), x.float() + d)
    h64 = h.cpu().double()
    H.check_blocks(t, h64 / torch.sqrt((h64 * h64).mean(-1, keepdim=True) + 1e-6) * w.double(), NORM_REL)


def test_norm_of_very_many_wide_rows(dev):
    """More rows of a width that takes a workgroup of 1024 threads each than one launch has threads for."""
    from pgmoe import exec_fused_rmsnorm_mx
    rows, cols = (1 << 22) + 5, 4128
    if torch.cuda.mem_get_info(dev)[0] < (rows * cols * 4):
        pytest.skip("needs 70 GB")
    x = torch.zeros(rows, cols, dtype=torch.float16, device=dev)
    at = torch.tensor([0, 1, (1 << 21) + 7, (1 << 22) - 2, (1 << 22) - 1, 1 << 22, rows - 1])
    some = _spread(len(at), cols, 14, torch.float16)
    x[at.to(dev)] = some.to(dev)
    w = torch.randn(cols, generator=torch.Generator().manual_seed(15)).to(dev)
    t = exec_fused_rmsnorm_mx(x, w)
    few = exec_fused_rmsnorm_mx(some.to(dev), w)
    assert torch.equal(t.codes[at.to(dev)], few.codes) and torch.equal(t.scales[at.to(dev)], few.scales)
    # the other rows are 0 w: zeros of w's sign
    assert not (t.codes[2:64] & 127).any() and not (t.codes[rows - 4:rows - 1] & 127).any()


def test_norm_rows_of_zeros_and_not_finite_ones(dev):
    from pgmoe import exec_fused_add_rmsnorm_mx
    x = torch.randn(6, 512, generator=torch.Generator().manual_seed(2))
    x[1] = 0
    x[2, 3], x[4, 500] = math.nan, math.inf
    x[5] *= 1e-20
    h, t = exec_fused_add_rmsnorm_mx(x.to(dev), torch.zeros(6, 512, device=dev), torch.ones(512, device=dev))
    e, v = H.scales(t), H.values(t)
    assert (e[1] == 0).all() and (v[1] == 0).all()
    assert (e[2] == 255).all() and (e[4, 15] == 255).all()
    assert (e[[0, 1, 3, 5]] != 255).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_more_chunks_than_one_launch_numbers(dev, fmt):
    """To blocks, back and the gated activation over 2^31 pieces of 16 bytes and more: rows on both sides of where calls are cut."""
    from pgmoe import exec_fused_act_mul_mx, mx_quantize
    rows, cols = (1 << 22) + 5, 4128
    if torch.cuda.mem_get_info(dev)[0] < rows * cols * 6:
        pytest.skip("needs 104 GB")
    cut = ((1 << 31) - 1) // (cols // 8)
    at = torch.tensor([0, 1, cut - 2, cut - 1, cut, cut + 1, rows - 1])
    x = torch.zeros(rows, cols, dtype=torch.float16, device=dev)
    some = _spread(len(at), cols, 19, torch.float16).to(dev)
    x[at.to(dev)] = some
    t, few = mx_quantize(x, fmt), mx_quantize(some, fmt)
    assert torch.equal(t.codes[at.to(dev)], few.codes) and torch.equal(t.scales[at.to(dev)], few.scales)
    assert not t.codes[cut + 2:cut + 64].any() and not t.codes[2:64].any()
    assert torch.equal(t.dequantize(torch.float16)[at.to(dev)], few.dequantize(torch.float16))
    del t
    t, few = exec_fused_act_mul_mx(x, x, "silu", fmt), exec_fused_act_mul_mx(some, some, "silu", fmt)
    assert torch.equal(t.codes[at.to(dev)], few.codes) and torch.equal(t.scales[at.to(dev)], few.scales)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 1440), (61, 768), (300, 4096)])
def test_act_mul(dev, fmt, act, dtype, rows, cols):
    from pgmoe import exec_fused_act_mul_mx
    g = torch.Generator().manual_seed(rows + cols)
    both = torch.randn(rows, 2 * cols, generator=g) * torch.exp(1.2 * torch.randn(rows, 2 * cols, generator=g))
    both = both.clamp(-90, 90).to(dtype)
    dv = both.to(dev)
    t = exec_fused_act_mul_mx(dv[:, :cols], dv[:, cols:], act, fmt)
    a, u = both[:, :cols].double(), both[:, cols:].double()
    if act == "silu":
        y = a / (1 + torch.exp(-a)) * u
    else:
        y = a / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3))) * u
    # beyond |g| of 90 in the exponent (the tanh form's cube) the fp32 value is zero: below 2^-126 of the block's rest
    H.check_blocks(t, torch.where(y.abs() < 1e-30, torch.zeros_like(y), y), ACT_REL)


# ---------------------------------------------------------------- product
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [
    (1, 1, 32), (1, 16, 128), (2, 17, 64), (5, 30, 96), (15, 100, 160), (16, 64, 512), (17, 257, 544), (33, 130, 1440),
    (64, 96, 2048), (65, 33, 288), (77, 1001, 1440), (130, 515, 320), (200, 256, 4096), (257, 300, 640), (1, 4099, 4096),
    (8, 2000, 8192), (300, 1030, 992), (520, 777, 1056), (1030, 513, 416),
    # enough outputs for the larger tiles, of 64, 128 and 256 rows
    (700, 4099, 96), (2001, 6000, 160), (4100, 8195, 64), (2050, 8190, 544)])
def test_product(dev, fmt, M, N, K):
    from pgmoe import HipMXLinear
    log(f"product {fmt} {M} x {N} x {K}")
    w, w64 = _random_blocks(N, K, "e2m1", N + K)
    x, x64 = _random_blocks(M, K, fmt, M + 3 * K)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(1)) * 100 if (M + N) % 2 else None
    layer = HipMXLinear(w, bias=None if bias is None else bias.to(dev))
    y, s = H.product(x64, w64, bias)
    for dt in (torch.float32, torch.bfloat16):
        out = layer(x, out_dtype=dt)
        assert out.dtype == dt and out.shape == (M, N)
        H.check_product(out, y, s, K, cut=fmt == "e4m3" and dt != torch.float32)


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("act_fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [(1, 100, 4096), (3, 1000, 96), (8, 48, 2080), (16, 272, 512), (17, 40, 672),
                                   (40, 33, 1440), (150, 300, 288)])
def test_product_of_values(dev, dtype, act_fmt, M, N, K):
    """Rows of floating-point values are brought to blocks first, whichever way the call does that."""
    from pgmoe import HipMXLinear, mx_quantize
    w, w64 = _random_blocks(N, K, "e2m1", N + K)
    x = _spread(M, K, M + K, dtype, span=1.0)
    layer = HipMXLinear(w, act_fmt=act_fmt)
    codes, e = H.encode(x, act_fmt)
    y, s = H.product(H.decode(codes, e, act_fmt), w64)
    out = layer((x * 0.01).to(dev), out_dtype=torch.float32)  # another call before, with other values
    out = layer(x.to(dev), out_dtype=torch.float32)
    H.check_product(out, y, s, K)
    assert torch.equal(out, layer(mx_quantize(x.to(dev), act_fmt), out_dtype=torch.float32))
    out = layer(x.to(dev).view(M, 1, K))
    assert out.shape == (M, 1, N) and out.dtype == dtype
    wide = torch.zeros(M, K + 64, dtype=dtype, device=dev)
    wide[:, 32:-32] = x.to(dev)
    assert torch.equal(layer(wide[:, 32:-32]).view(M, 1, N), out)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K,dtype", [((1 << 20) + 9, 48, 8224, torch.float32), ((1 << 20) + 9, 2100, 96, torch.float16),
                                         (3, (1 << 21) + 7, 4128, torch.float16), (21, (1 << 21) + 7, 4128, torch.float32)])
def test_product_of_far_offsets(dev, fmt, M, N, K, dtype):
    """Blocks, weights and outputs whose bytes pass 2^32 and whose outputs pass 2^31."""
    from pgmoe import HipMXLinear, MXTensor
    if torch.cuda.mem_get_info(dev)[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    g = torch.Generator(device=dev).manual_seed(M + N)

    def blocks(rows, f):
        codes = torch.randint(0, 256, (rows, K if f == "e4m3" else K // 2), generator=g, device=dev, dtype=torch.uint8)
        if f == "e4m3":
            codes.masked_fill_(codes & 127 == 127, 0)
        return MXTensor(codes, torch.randint(118, 124, (rows, K // 32), generator=g, device=dev, dtype=torch.uint8), f)

    def some(t, at):
        at = at.to(dev)
        return H.values(MXTensor(t.codes[at], t.scales[at], t.fmt))

    x, w = blocks(M, fmt), blocks(N, "e2m1")
    out = HipMXLinear(w)(x, out_dtype=dtype)
    pick = lambda n: torch.unique(torch.tensor([0, 1, n // 2, n - 9, n - 2, n - 1]).clamp(min=0))  # noqa: E731
    m, n = pick(M), pick(N)
    y, s = H.product(some(x, m), some(w, n))
    H.check_product(out[m.to(dev)][:, n.to(dev)], y, s, K, cut=fmt == "e4m3" and dtype != torch.float32)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("N", [8160, 8177, 8209])
def test_product_of_few_long_rows(dev, fmt, N):
    """Rows of more than 4096 against outputs that a workgroup takes 16 or 32 of at a time."""
    from pgmoe import HipMXLinear
    for M, K in [(1, 4128), (7, 6176), (16, 8192)]:
        w, w64 = _random_blocks(N, K, "e2m1", N + M)
        x, x64 = _random_blocks(M, K, fmt, M)
        y, s = H.product(x64, w64)
        H.check_product(HipMXLinear(w)(x, out_dtype=torch.float32), y, s, K)


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("act_fmt", FMTS)
@pytest.mark.parametrize("K", [32, 96, 512, 1440, 2048, 2080, 4064, 4096, 4128, 8224])
def test_product_of_few_rows_of_values(dev, dtype, act_fmt, K):
    """Every number of rows that become blocks inside the product, and rows too long for that: the same bits as by two calls;
    one of them with a block that is not finite."""
    from pgmoe import HipMXLinear, mx_quantize
    w, _ = _random_blocks(70, K, "e2m1", K)
    layer = HipMXLinear(w, act_fmt=act_fmt)
    x = _spread(16, K, K + 1, dtype, span=1.0)
    x[3, K - 1], x[9, 0] = float("inf"), float("nan")
    x = x.to(dev)
    for M in range(1, 17):
        got, want = layer(x[:M], out_dtype=torch.float32), layer(mx_quantize(x[:M], act_fmt), out_dtype=torch.float32)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num()), M
        assert torch.equal(got.isnan().all(1).cpu(), torch.arange(M).eq(3) | torch.arange(M).eq(9)) and not got[:3].isnan().any()


@pytest.mark.parametrize("fmt,dtype", [("e4m3", torch.float32), ("e4m3", torch.float16), ("e2m1", torch.float32)])
@pytest.mark.parametrize("K", [32, 512, 544, 1056, 1536, 2080, 4128])
def test_product_of_few_tiles(dev, fmt, dtype, K):
    """The inputs shared out among parts of a workgroup, some of which have fewer or none."""
    from pgmoe import HipMXLinear
    for M, N in [(17, 16), (40, 70), (65, 130), (90, 300), (260, 520)]:
        w, w64 = _random_blocks(N, K, "e2m1", M + K)
        x, x64 = _random_blocks(M, K, fmt, M)
        layer = HipMXLinear(w, bias=torch.arange(N, dtype=torch.float32, device=dev))
        y, s = H.product(x64, w64, torch.arange(N))
        out = layer(x, out_dtype=dtype)
        assert torch.equal(layer(x, out_dtype=dtype), out)
        # sums of 65520 and more, half a step past the largest, are infinities in fp16: those within the sum's own error
        # (as in check_product, before its rounding) of that may be
        over = torch.isinf(out.cpu())
        error = (K / 128 + 17) * 2.0 ** -21 * s[0] + 2.0 ** -10 * s[1]
        assert not over.any() or dtype == torch.float16
        assert (y.abs() + error)[over].ge(65520).all() and torch.equal(out.cpu()[over] > 0, y[over] > 0)
        out, y = out.cpu().masked_fill(over, 0), y.masked_fill(over, 0)
        H.check_product(out, y, s, K, cut=fmt == "e4m3" and dtype != torch.float32)


def test_product_exact_sums(dev):
    """Small whole numbers: every order of the sum is exact, so every output is, in each way the work is laid out."""
    from pgmoe import HipMXLinear, MXTensor
    for M, N, K in [(1, 50, 512), (13, 129, 1120), (50, 300, 1440), (100, 257, 2016), (333, 700, 800), (700, 1300, 544)]:
        g = torch.Generator().manual_seed(M)
        wc, xc = torch.randint(0, 16, (N, K), generator=g), torch.randint(0, 16, (M, K), generator=g)
        one = torch.full((1, K // 32), 128, dtype=torch.uint8)
        w = MXTensor(H.pack(wc, "e2m1").to(dev), one.expand(N, -1).to(dev), "e2m1")
        x4 = MXTensor(H.pack(xc, "e2m1").to(dev), one.expand(M, -1).to(dev), "e2m1")
        v = H.decode(xc, one.long().expand(M, -1), "e2m1")
        ref = v @ H.decode(wc, one.long().expand(N, -1), "e2m1").T
        x8 = MXTensor(v.float().div(2).to(torch.float8_e4m3fn).to(dev), one.to(dev).expand(M, -1), "e4m3")
        layer = HipMXLinear(w)
        assert torch.equal(layer(x4, out_dtype=torch.float32).cpu().double(), ref), (M, N, K)
        assert torch.equal(layer(x8, out_dtype=torch.float32).cpu().double(), ref), (M, N, K)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M", [1, 20, 70, 300])
def test_product_of_nan_blocks(dev, fmt, M):
    """A NaN block of a row (of weights) makes that row (column) of the output NaN and no other; far scales."""
    from pgmoe import HipMXLinear, MXTensor
    N, K = 90, 416
    w, _ = _random_blocks(N, K, "e2m1", 4)
    x, _ = _random_blocks(M, K, fmt, 5)
    ws, xs = w.scales.clone(), x.scales.clone()
    ws[17, 12], xs[M // 2, 0], xs[M - 1, 12] = 255, 255, 255
    w, x = MXTensor(w.codes, ws, "e2m1"), MXTensor(x.codes, xs, fmt)
    out = torch.isnan(HipMXLinear(w)(x, out_dtype=torch.float32)).cpu()
    want = torch.zeros(M, N, dtype=torch.bool)
    want[M // 2], want[M - 1], want[:, 17] = True, True, True
    assert torch.equal(out, want)


@pytest.mark.parametrize("M", [1, 16, 20, 70, 300])
def test_product_of_nan_codes(dev, M):
    """The e4m3 codes 0x7f and 0xff are NaN, whatever their block's scale."""
    from pgmoe import HipMXLinear, MXTensor
    N, K = 70, 416
    w, _ = _random_blocks(N, K, "e2m1", 4)
    x, _ = _random_blocks(M, K, "e4m3", 5)
    c = x.codes.clone()
    c[M // 2, 3], c[M - 1, K - 1] = 0x7f, 0xff
    x = MXTensor(c, x.scales, "e4m3")
    want = torch.zeros(M, dtype=torch.bool)
    want[M // 2], want[M - 1] = True, True
    assert torch.equal(torch.isnan(x.dequantize().cpu()).any(1), want)
    for dt in H.DTYPES:
        assert torch.equal(torch.isnan(HipMXLinear(w)(x, out_dtype=dt)).cpu(), want[:, None].expand(M, N)), dt


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M", [1, 16, 20, 70, 300])
@pytest.mark.parametrize("xs,ws", [(3, 250), (10, 244), (30, 210), (130, 110), (240, 24), (246, 3)])
def test_product_of_far_scales(dev, fmt, M, xs, ws):
    """Rows near the ends of fp32's normal range against weights near the other end: nothing is lost on the way."""
    from pgmoe import HipMXLinear
    N, K = 90, 288
    w, w64 = _random_blocks(N, K, "e2m1", 12, ws, ws + 1)
    x, x64 = _random_blocks(M, K, fmt, 13, xs, xs + 1)
    y, s = H.product(x64, w64)
    for dt in (torch.float32, torch.bfloat16):
        H.check_product(HipMXLinear(w)(x, out_dtype=dt), y, s, K, cut=fmt == "e4m3" and dt != torch.float32)


def test_product_takes_views_of_blocks(dev):
    from pgmoe import HipMXLinear, MXTensor
    w, w64 = _random_blocks(40, 128, "e2m1", 7)
    layer = HipMXLinear(w)
    for fmt in FMTS:
        x, x64 = _random_blocks(60, 512, fmt, 8)
        half = 64 if fmt == "e2m1" else 128
        for rows, at in ((slice(None), 0), (slice(3, 50, 2), 1), (slice(9, 10), 2)):
            v = MXTensor(x.codes[rows, at * half:(at + 1) * half], x.scales[rows, 4 * at:4 * at + 4], fmt)
            y, s = H.product(x64[rows, 128 * at:128 * at + 128], w64)
            H.check_product(layer(v, out_dtype=torch.float32), y, s, 128)
    x, _ = _random_blocks(60, 128, "e4m3", 9)
    assert layer(MXTensor(x.codes.view(3, 4, 5, 128), x.scales.view(3, 4, 5, 4), "e4m3")).shape == (3, 4, 5, 40)
    assert layer(MXTensor(x.codes[:0], x.scales[:0], "e4m3")).shape == (0, 40)


@pytest.mark.parametrize("fmt", FMTS)
def test_room_between_rows_is_left_alone(dev, fmt):
    """Blocks written at strides of the caller's: nothing lands between the rows, before or behind them."""
    import ctypes
    from pgmoe import exec_fused_act_mul_mx, exec_fused_rmsnorm_mx, mx_quantize
    from pgmoe._lib import Mx, check, lib
    st = torch.cuda.current_stream().cuda_stream
    for rows, cols in [(1, 32), (3, 96), (70, 544), (9, 4128)]:
        n, bits = cols if fmt == "e4m3" else cols // 2, 8 if fmt == "e4m3" else 4
        cs, ss = (n + 15) // 16 * 16 + 32, (cols // 32 + 15) // 16 * 16 + 16
        x = _spread(rows, cols, 20, torch.float16).to(dev)
        w = torch.randn(cols, generator=torch.Generator().manual_seed(21)).to(dev)
        calls = [(mx_quantize(x, fmt), lambda y: lib().pgmoe_mx_quantize(x.data_ptr(), 1, cols, y, st)),
                 (exec_fused_act_mul_mx(x, x, "gelu", fmt),
                  lambda y: lib().pgmoe_mx_act_mul(x.data_ptr(), cols, x.data_ptr(), cols, 1, 1, y, st)),
                 (exec_fused_rmsnorm_mx(x, w, 1e-6, fmt),
                  lambda y: lib().pgmoe_add_rmsnorm_mx(x.data_ptr(), 1, None, 0, w.data_ptr(), 1e-6, None, y, st))]
        for want, call in calls:
            codes = torch.full((rows + 2, cs), 0x5a, dtype=torch.uint8, device=dev)
            scales = torch.full((rows + 2, ss), 0x5a, dtype=torch.uint8, device=dev)
            y = Mx(codes[1].data_ptr(), scales[1].data_ptr(), cs, ss, rows, cols, bits)
            check(call(ctypes.byref(y)), "call")
            torch.cuda.synchronize()
            assert torch.equal(codes[1:-1, :n], want.codes) and torch.equal(scales[1:-1, :cols // 32], want.scales)
            codes[1:-1, :n], scales[1:-1, :cols // 32] = 0x5a, 0x5a
            assert (codes == 0x5a).all() and (scales == 0x5a).all()


def test_outputs_past_the_end_are_left_alone(dev):
    """Ragged outputs written into the middle of a larger buffer, through the C ABI."""
    from pgmoe import HipMXLinear
    from pgmoe._lib import check, lib
    for M, N, K in [(1, 1, 32), (3, 5, 64), (17, 33, 96), (70, 130, 160), (130, 257, 288), (300, 515, 512)]:
        w, w64 = _random_blocks(N, K, "e2m1", 1)
        x, x64 = _random_blocks(M, K, "e4m3", 2)
        layer = HipMXLinear(w)
        buf = torch.full((M * N + 512,), 7.0, device=dev)
        out = buf[256:256 + M * N]
        check(lib().pgmoe_mx_linear(layer._packed.data_ptr(), N, x._ref, None, out.data_ptr(), 0,
                                    torch.cuda.current_stream().cuda_stream), "pgmoe_mx_linear")
        torch.cuda.synchronize()
        assert (buf[:256] == 7).all() and (buf[256 + M * N:] == 7).all()
        y, s = H.product(x64, w64)
        H.check_product(out, y, s, K)


# ---------------------------------------------------------------- weights of GGUF files
def test_from_gguf_keeps_mxfp4_exactly(dev):
    from pgmoe import HipMXLinear
    rng = np.random.default_rng(3)
    rows, cols = 70, 320
    raw = rng.integers(0, 256, (rows, cols // 32, 17), dtype=np.uint8)
    raw[..., 0] = rng.integers(118, 130, (rows, cols // 32))
    codes = torch.from_numpy(np.concatenate((raw[..., 1:] & 15, raw[..., 1:] >> 4), -1).astype(np.int64)).reshape(rows, cols)
    w64 = H.decode(codes, torch.from_numpy(raw[..., 0].astype(np.int64)), "e2m1")
    f = torch.randn(30, cols, generator=torch.Generator().manual_seed(1))
    gguf = _gguf({"a.weight": (39, (rows, cols), raw.tobytes()), "b.weight": (0, (30, cols), f.numpy().tobytes())})
    x, x64 = _random_blocks(9, cols, "e4m3", 6)
    layer = HipMXLinear.from_gguf(gguf, "a.weight", device=dev)
    y, s = H.product(x64, w64)
    H.check_product(layer(x, out_dtype=torch.float32), y, s, cols)
    c, e = H.encode(f, "e2m1")
    both = HipMXLinear.from_gguf(gguf, ["a.weight", "b.weight"], device=dev)
    y, s = H.product(x64, torch.cat((w64, H.decode(c, e, "e2m1"))))
    H.check_product(both(x, out_dtype=torch.float32), y, s, cols)


def _gguf(tensors):
    """The reader's surface over bytes in memory."""
    class Info:
        def __init__(self, qtype, shape):
            self.qtype, self.shape = qtype, shape

    class File:
        def __init__(self):
            self.tensors = {n: Info(q, s) for n, (q, s, _) in tensors.items()}

        def get_tensor_bytes(self, name):
            return np.frombuffer(tensors[name][2], dtype=np.uint8)

    return File()


# ---------------------------------------------------------------- as they are used
def test_ffn_of_blocks(dev):
    """Norm, gate and up product, activation, down product: each step against float64 of the step's own input."""
    from pgmoe import HipMXLinear, exec_fused_act_mul_mx, exec_fused_add_rmsnorm_mx, mx_quantize
    D, I = 512, 800
    g = torch.Generator().manual_seed(4)
    gu = HipMXLinear(mx_quantize((0.05 * torch.randn(2 * I, D, generator=g)).to(dev), "e2m1"))
    down_w = mx_quantize((0.05 * torch.randn(D, I, generator=g)).to(dev), "e2m1")
    down = HipMXLinear(down_w)
    w = (1 + 0.1 * torch.randn(D, generator=g)).to(dev)
    for M in (1, 6, 40, 300):
        x, delta = torch.randn(M, D, generator=g).to(dev), torch.randn(M, D, generator=g).to(dev)
        h, n = exec_fused_add_rmsnorm_mx(x, delta, w)
        y = gu(n, out_dtype=torch.float16)
        a = exec_fused_act_mul_mx(y[:, :I], y[:, I:])
        y64 = y.double().cpu()
        H.check_blocks(a, y64[:, :I] / (1 + torch.exp(-y64[:, :I])) * y64[:, I:], ACT_REL)
        out = down(a, out_dtype=torch.float32)
        H.check_product(out, *H.product(H.values(a), H.values(down_w)), I)


def test_other_streams_and_graphs(dev):
    """The run on another stream, and replayed from graphs: two of one layer, in turn, with eager calls between."""
    from pgmoe import HipMXLinear, exec_fused_act_mul_mx, exec_fused_add_rmsnorm_mx, mx_quantize
    D, I = 256, 320
    g = torch.Generator().manual_seed(6)
    gu = HipMXLinear(mx_quantize((0.1 * torch.randn(2 * I, D, generator=g)).to(dev), "e2m1"))
    down = HipMXLinear(mx_quantize((0.1 * torch.randn(D, I, generator=g)).to(dev), "e2m1"))
    w = torch.ones(D, device=dev)

    def step(x, delta):
        h, n = exec_fused_add_rmsnorm_mx(x, delta, w)
        y = gu(n)
        return h + down(exec_fused_act_mul_mx(y[:, :I], y[:, I:]), out_dtype=torch.float32) + down(y[:, :I], out_dtype=torch.float32)

    for M in (1, 90):
        draw = lambda: (torch.randn(M, D, generator=g).to(dev), torch.randn(M, D, generator=g).to(dev))  # noqa: E731
        inputs = [draw() for _ in range(4)]
        ref = [step(*i).clone() for i in inputs]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = [step(*i) for i in inputs]
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(again, ref))
        static = [draw(), draw()]
        graphs, outs = [], []
        for s in static:
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                outs.append(step(*s))
            graphs.append(gr)
        for turn in range(3):
            for k in (0, 1):
                i = (turn + k) % 4
                for d, v in zip(static[k], inputs[i]):
                    d.copy_(v)
                graphs[k].replay()
                step(*inputs[(i + 1) % 4])
                torch.cuda.synchronize()
                assert torch.equal(outs[k], ref[i])


def test_same_bits_again(dev):
    """No order of sums depends on the run, nor on the other rows of a call of the same size."""
    from pgmoe import HipMXLinear
    w, _ = _random_blocks(300, 1440, "e2m1", 1)
    layer = HipMXLinear(w)
    for M in (4, 50, 200):
        x, _ = _random_blocks(M, 1440, "e4m3", 2)
        first = layer(x, out_dtype=torch.float32)
        for _ in range(3):
            assert torch.equal(layer(x, out_dtype=torch.float32), first)


# ---------------------------------------------------------------- what is refused
def test_refusals(dev):
    from pgmoe import HipMXLinear, MXTensor, exec_fused_act_mul_mx, exec_fused_add_rmsnorm_mx, exec_fused_rmsnorm_mx, mx_quantize
    x = torch.randn(4, 64, device=dev)
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=dev)  # noqa: E731
    w = mx_quantize(torch.randn(8, 64, device=dev), "e2m1")
    layer = HipMXLinear(w)
    for err, call in [
            (ValueError, lambda: mx_quantize(x[:, :48])), (NotImplementedError, lambda: mx_quantize(x, "e5m2")),
            (NotImplementedError, lambda: mx_quantize(x.double())), (NotImplementedError, lambda: mx_quantize(x).dequantize(torch.int8)),
            (ValueError, lambda: exec_fused_rmsnorm_mx(x, torch.ones(32, device=dev))),
            (ValueError, lambda: exec_fused_rmsnorm_mx(x, torch.ones(64, device=dev), -1.0)),
            (ValueError, lambda: exec_fused_add_rmsnorm_mx(x, x[:2], torch.ones(64, device=dev))),
            (NotImplementedError, lambda: exec_fused_add_rmsnorm_mx(x, x.double(), torch.ones(64, device=dev))),
            (NotImplementedError, lambda: exec_fused_act_mul_mx(x, x, "relu")), (ValueError, lambda: exec_fused_act_mul_mx(x, x[:2])),
            (ValueError, lambda: exec_fused_act_mul_mx(x, x.half())), (ValueError, lambda: MXTensor(u8(4, 64), u8(4, 3))),
            (ValueError, lambda: MXTensor(u8(4, 48), u8(4, 1))), (ValueError, lambda: MXTensor(x, u8(4, 2))),
            (ValueError, lambda: MXTensor(u8(4, 64), x[:, :2])), (NotImplementedError, lambda: MXTensor(u8(4, 64), u8(4, 2), "e3m2")),
            (ValueError, lambda: HipMXLinear(mx_quantize(x))), (ValueError, lambda: HipMXLinear(w, bias=torch.zeros(9, device=dev))),
            (ValueError, lambda: HipMXLinear(mx_quantize(x[0], "e2m1"))), (NotImplementedError, lambda: HipMXLinear(w, act_fmt="f16")),
            (ValueError, lambda: layer(x[:, :32])), (NotImplementedError, lambda: layer(x, out_dtype=torch.float64)),
            (ValueError, lambda: layer(x.cpu())), (NotImplementedError, lambda: layer(x.double(), out_dtype=torch.float32)),
            (NotImplementedError, lambda: HipMXLinear.from_gguf(_gguf({"a": (12, (4, 256), b"")}), "a", device=dev)),
            (ValueError, lambda: HipMXLinear.from_gguf(_gguf({"a": (0, (4, 48), b"")}), "a", device=dev)),
            (ValueError, lambda: HipMXLinear.from_gguf(_gguf({"a": (39, (2, 4, 32), bytes(136))}), "a", device=dev)),
            (ValueError, lambda: HipMXLinear.from_gguf(_gguf({"a": (0, (32,), bytes(128))}), "a", device=dev)),
            (KeyError, lambda: HipMXLinear.from_gguf(_gguf({}), "a", device=dev))]:
        with pytest.raises(err):
            call()
