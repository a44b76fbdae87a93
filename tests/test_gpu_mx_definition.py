"""Microscaled operators against the float64 formulas where roundings on the way would show: codes next to borders, values
near the ends of fp32's range."""

import pytest

import mx_helpers as H

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FMTS = ["e4m3", "e2m1"]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda", 0)


# ---------------------------------------------------------------- norm
def _norm64(h, w, eps):
    return h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


@pytest.mark.parametrize("fmt,rows,cols,dt,ddt", [
    ("e4m3", 2000, 4096, torch.float32, torch.float16), ("e2m1", 2000, 4096, torch.float32, torch.float32),
    ("e4m3", 700, 8192, torch.bfloat16, torch.float32), ("e4m3", 3000, 1024, torch.float16, None),
    ("e4m3", 100, 20000, torch.float32, torch.bfloat16), ("e2m1", 9000, 224, torch.float32, None), ("e4m3", 500, 4064, torch.float32, None)])
def test_norm_codes_are_the_formulas(dev, fmt, rows, cols, dt, ddt):
    """Every code and scale byte of millions: nothing is rounded before them but to 64 bits."""
    from pgmoe import exec_fused_add_rmsnorm_mx, exec_fused_rmsnorm_mx
    g = torch.Generator().manual_seed(rows + cols)
    x = (3 * torch.randn(rows, cols, generator=g) * torch.exp(0.5 * torch.randn(cols, generator=g))).to(dt)
    w = 1 + 0.2 * torch.randn(cols, generator=g)
    h = x.double()
    if ddt is None:
        t = exec_fused_rmsnorm_mx(x.to(dev), w.to(dev), 1e-6, fmt)
    else:
        d = torch.randn(rows, cols, generator=g).to(ddt)
        h = h + d.double()
        got, t = exec_fused_add_rmsnorm_mx(x.to(dev), d.to(dev), w.to(dev), 1e-6, fmt)
        assert torch.equal(got.cpu(), h.float())
    codes, e = H.encode(_norm64(h, w, float(torch.tensor(1e-6))), fmt)  # eps as the C ABI takes it, in fp32
    assert torch.equal(H.scales(t), e)
    assert torch.equal(H.unpack(t), codes)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("cols", [64, 512, 2048, 4096, 8192, 16512])
def test_norm_of_far_rows(dev, fmt, cols):
    """Rows whose squares are beyond fp32's range, or below it with nothing added."""
    from pgmoe import exec_fused_add_rmsnorm_mx, exec_fused_rmsnorm_mx
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(6, cols, generator=g) * torch.tensor([1e25, 5e37, 1e-25, 1e-37, 1.0, 1e19])[:, None]
    w = 1 + 0.2 * torch.randn(cols, generator=g)
    for eps in (0.0, 1e-6):
        codes, e = H.encode(_norm64(x.double(), w, float(torch.tensor(eps))), fmt)
        t = exec_fused_rmsnorm_mx(x.to(dev), w.to(dev), eps, fmt)
        h, u = exec_fused_add_rmsnorm_mx(x.to(dev), torch.zeros_like(x).to(dev), w.to(dev), eps, fmt)
        assert torch.equal(h.cpu(), x)
        for v in (t, u):
            assert torch.equal(H.scales(v), e) and torch.equal(H.unpack(v), codes)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("cols", [96, 4096, 16512])
def test_norm_of_far_weights(dev, fmt, cols):
    """Rows that end below fp32's normal range, or beyond it; sums that only h does not hold."""
    from pgmoe import exec_fused_add_rmsnorm_mx, exec_fused_rmsnorm_mx
    g = torch.Generator().manual_seed(cols)
    x, w = torch.randn(5, cols, generator=g), 1 + 0.2 * torch.randn(cols, generator=g)
    for size in (2.0 ** -120, 2.0 ** -128, 2.0 ** -133, 2.0 ** 120):
        y = _norm64(x.double(), w * size, float(torch.tensor(1e-6)))
        # below 2^-126 a value is rounded to 2^-149 first: 2^-14 of the codes' least half step
        H.check_blocks(exec_fused_rmsnorm_mx(x.to(dev), (w * size).to(dev), 1e-6, fmt), y, 2.0 ** -11)
    t = exec_fused_rmsnorm_mx(x.to(dev), torch.full((cols,), 3e38, device=dev), 1e-6, fmt)
    over = _norm64(x.double(), torch.full((cols,), 3e38), 1e-6).abs().ge(2.0 ** 128).reshape(5, -1, 32).any(-1)
    assert torch.equal(H.scales(t) == 255, over)
    big = torch.full((5, cols), 3e38).copysign(x)
    h, t = exec_fused_add_rmsnorm_mx(big.to(dev), big.to(dev), w.to(dev), 1e-6, fmt)
    codes, e = H.encode(_norm64(2 * big.double(), w, 1e-6), fmt)
    assert torch.isinf(h).all() and torch.equal(H.scales(t), e) and torch.equal(H.unpack(t), codes)


# ---------------------------------------------------------------- activation
def _act64(act, g, u):
    if act == "silu":
        return g / (1 + torch.exp(-g)) * u
    return g / (1 + torch.exp(-2 * (2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3))) * u


# what fp32 leaves of a product: 2^-23 each of a power of two and a reciprocal, four roundings and what the first order leaves
# out; of gelu's exponent eight roundings of 2^-24, times its size, up to 400 ln 2
_FAR_REL = {"silu": 2.0 ** -20, "gelu": 2.0 ** -12}


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("act,lo,hi,size", [
    ("silu", -84, -60, 1.0), ("silu", -105, -82, 1e20), ("silu", -180, -90, 3e38), ("silu", -400, -170, 3e38), ("silu", -90, 90, 1e30),
    ("gelu", -8, -5, 1.0), ("gelu", -10.5, -8, 1e20), ("gelu", -14, -9.5, 3e38), ("gelu", -30, -12, 3e38), ("gelu", -14, 14, 1e30)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_act_of_far_gates(dev, fmt, act, lo, hi, size, dtype):
    """Negative gates whose activation is far below one, beside values that bring the product back."""
    from pgmoe import exec_fused_act_mul_mx
    gen = torch.Generator().manual_seed(int(-lo) + len(act))
    g = (lo + (hi - lo) * torch.rand(130, 320, generator=gen)).to(dtype)
    u = (size * (0.01 + 0.99 * torch.rand(130, 320, generator=gen))).clamp(max=3.3e38).to(dtype)
    g[:3] = torch.tensor([lo, (lo + hi) / 2, hi]).to(dtype)[:, None]
    t = exec_fused_act_mul_mx(g.to(dev), u.to(dev), act, fmt)
    y = _act64(act, g.double(), u.double())
    H.check_blocks(t, torch.where(y.abs() < 2.0 ** -140, torch.zeros_like(y), y), _FAR_REL[act])


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_act_of_the_largest_gates(dev, act):
    """Gates at both ends of fp32's range: the gate itself, or nothing; not finite ones make NaN blocks."""
    from pgmoe import exec_fused_act_mul_mx
    top = torch.finfo(torch.float32).max
    g = torch.tensor([top, -top, 1e30, -1e30, 1e10, -1e10, -1000.0, float("inf"), -float("inf"), float("nan")])[:, None].repeat(1, 32)
    u = torch.full_like(g, 0.5)
    t = exec_fused_act_mul_mx(g.to(dev), u.to(dev), act)
    v = t.dequantize().cpu()
    want, _ = H.encode(torch.where(g > 0, g * 0.5, torch.zeros_like(g))[:7], "e4m3")
    assert torch.equal(H.unpack(t)[:7] & 127, want)
    assert torch.isfinite(v[:7]).all() and torch.isnan(v[7:]).all()


# ---------------------------------------------------------------- product
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M", [1, 5, 16, 20, 70])
@pytest.mark.parametrize("K", [32, 288, 512, 544, 2080, 4128, 8224])
def test_product_of_infinite_blocks(dev, fmt, M, K):
    """Blocks beyond fp32's range, the row's last among them: sums of one sign are infinite, and other rows as they were."""
    from pgmoe import HipMXLinear, MXTensor
    N = 40
    g = torch.Generator().manual_seed(K + M)
    wc = torch.randint(1, 8, (N, K), generator=g)
    top = 8 if fmt == "e2m1" else 127
    xc = torch.randint(1, top, (M, K), generator=g)
    ws, xs = torch.full((N, K // 32), 127), torch.full((M, K // 32), 120)
    far = sorted({0, M // 2, M - 1})
    if fmt == "e4m3":
        xc[far, -32:] = torch.randint(80, top, (len(far), 32), generator=g)
    for i, r in enumerate(far):
        xs[r, -1 if i != 1 else 0] = 254
        if i == 1:
            xc[r, :32] = top - 1
    w = MXTensor(H.pack(wc, "e2m1").to(dev), ws.to(torch.uint8).to(dev), "e2m1")
    x = MXTensor(H.pack(xc, fmt).to(dev), xs.to(torch.uint8).to(dev), fmt)
    y = H.decode(xc, xs, fmt) @ H.decode(wc, ws, "e2m1").T
    assert (y[far] > 2.0 ** 129).all()
    for dt in H.DTYPES:
        out = HipMXLinear(w)(x, out_dtype=dt).cpu()
        assert (out[far] == float("inf")).all(), dt
        rest = [r for r in range(M) if r not in far]
        torch.testing.assert_close(out[rest].double(), y[rest], rtol=2.0 ** -7, atol=0)


def _random_blocks(rows, cols, fmt, seed, dev):
    """Any codes but NaN, scales within 2^14 of each other."""
    from pgmoe import MXTensor
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256 if fmt == "e4m3" else 16, (rows, cols), generator=g)
    if fmt == "e4m3":
        codes = torch.where(codes % 128 == 127, torch.zeros_like(codes), codes)
    e = torch.randint(117, 131, (rows, cols // 32), generator=g)
    return MXTensor(H.pack(codes, fmt).to(dev), e.to(torch.uint8).to(dev), fmt), H.decode(codes, e, fmt)


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("act_fmt", FMTS)
@pytest.mark.parametrize("M,K", [(2, 512), (5, 96), (8, 4096), (9, 1440), (16, 2080), (16, 4096), (50, 1440), (200, 544)])
def test_rows_do_not_depend_on_the_others(dev, dtype, act_fmt, M, K):
    """Rows of values in another order, and one row among others of other values: the same bits for each row."""
    from pgmoe import HipMXLinear
    layer = HipMXLinear(_random_blocks(300, K, "e2m1", K, dev)[0], act_fmt=act_fmt)
    g = torch.Generator().manual_seed(M)
    x = (torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).to(dtype).to(dev)
    order = torch.randperm(M, generator=g).to(dev)
    for dt in (torch.float32, torch.float16):
        out = layer(x, out_dtype=dt)
        assert torch.equal(layer(x[order], out_dtype=dt), out[order])
        for i in (0, M // 2, M - 1):
            other = torch.randn(M, K, generator=g).to(dtype).to(dev)
            other[i] = x[i]
            assert torch.equal(layer(other, out_dtype=dt)[i], out[i])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 32), (3, 5, 64), (16, 515, 96), (17, 33, 96), (70, 130, 160), (130, 257, 288), (300, 515, 512),
                                   (700, 4099, 96), (2050, 8190, 64), (4100, 8195, 64), (3, 8209, 4128)])
def test_outputs_past_the_end_are_left_alone(dev, fmt, dtype, M, N, K):
    """Whole and ragged tiles of every size, written into the middle of a larger buffer through the C ABI."""
    from pgmoe import HipMXLinear
    from pgmoe._lib import check, lib
    w, w64 = _random_blocks(N, K, "e2m1", 1, dev)
    x, x64 = _random_blocks(M, K, fmt, 2, dev)
    layer = HipMXLinear(w)
    buf = torch.full((M * N + 1024,), 7.0, device=dev, dtype=dtype)
    out = buf[512:512 + M * N]
    check(lib().pgmoe_mx_linear(layer._packed.data_ptr(), N, x._ref, None, out.data_ptr(), {torch.float32: 0, torch.float16: 1}.get(dtype, 30),
                                torch.cuda.current_stream().cuda_stream), "pgmoe_mx_linear")
    torch.cuda.synchronize()
    assert (buf[:512] == 7).all() and (buf[512 + M * N:] == 7).all()
    at = torch.unique(torch.tensor([0, 1, M // 2, M - 2, M - 1]).clamp(0, M - 1))
    got = out.view(M, N)[at.to(dev)]
    y, s = H.product(x64[at], w64)
    over = y.abs() > 6e4  # fp16 ends there
    got = got.masked_fill(over.to(dev), 0) if dtype == torch.float16 else got
    y = y.masked_fill(over, 0) if dtype == torch.float16 else y
    H.check_product(got, y, s, K, cut=fmt == "e4m3" and dtype != torch.float32)


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("M,N,K", [(3, 100, 1440), (17, 33, 96), (70, 130, 4096), (300, 1030, 992), (700, 2050, 544), (2050, 4099, 160)])
def test_product_of_fp32_sums(dev, dtype, M, N, K):
    """Outputs of any type without the 8-bit products' cut, from blocks and from values, with a bias."""
    from pgmoe import HipMXLinear, MXTensor
    w, w64 = _random_blocks(N, K, "e2m1", N + K, dev)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(1)) * 10
    layer = HipMXLinear(w, bias=bias.to(dev), fp32_sums=True)
    x, x64 = _random_blocks(M, K, "e4m3", M + K, dev)
    y, s = H.product(x64 / 64, w64 / 64, bias)  # within fp16's range
    layer_small = HipMXLinear(MXTensor(w.codes, w.scales - 6, "e2m1"), bias=bias.to(dev), fp32_sums=True)
    H.check_product(layer_small(MXTensor(x.codes, x.scales - 6, "e4m3"), out_dtype=dtype), y, s, K)
    v = torch.randn(M, K, generator=torch.Generator().manual_seed(2)).to(dtype)
    codes, e = H.encode(v, "e4m3")
    y, s = H.product(H.decode(codes, e, "e4m3"), w64, bias)
    H.check_product(layer(v.to(dev), out_dtype=torch.float32), y, s, K)
    assert torch.equal(layer(v.to(dev), out_dtype=torch.float32), HipMXLinear(w, bias=bias.to(dev))(v.to(dev), out_dtype=torch.float32))


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("M", [1, 16, 17, 80, 300, 2100])
def test_fp32_sums_keep_small_products_beside_large_ones(dev, dtype, M):
    """Two products that cancel out, 15 octaves above the others: in a call of any number of rows the others' sum is exact."""
    from pgmoe import HipMXLinear, MXTensor
    N, K = 130, 32
    x, w = torch.full((M, K), 2.0 ** -4), torch.full((N, K), 2, dtype=torch.long)  # codes of 1
    x[:, 0], x[:, 8] = 448, 448
    w[:, 0], w[:, 8] = 7, 15  # 6 and -6
    one = torch.full((1, 1), 127, dtype=torch.uint8, device=dev)
    xt = MXTensor(x.to(torch.float8_e4m3fn).to(dev), one.expand(M, 1), "e4m3")
    wt = MXTensor(H.pack(w, "e2m1").to(dev), one.expand(N, 1), "e2m1")
    out = HipMXLinear(wt, fp32_sums=True)(xt, out_dtype=dtype)
    assert torch.equal(out, torch.full((M, N), 30 * 2.0 ** -4, dtype=dtype, device=dev))


# ---------------------------------------------------------------- calls
def test_wide_rows_are_not_copied(dev):
    """Rows of 16 MB, next to each other and of a wider matrix: read where they are, as narrow ones."""
    from pgmoe import HipMXLinear, exec_fused_act_mul_mx, exec_fused_rmsnorm_mx, mx_quantize
    base = torch.randn(5, 1 << 22, generator=torch.Generator().manual_seed(3)).to(dev)
    w = torch.ones(1 << 22, device=dev)
    part, few = base[:, 4096:8192], base[:, 4096:8192].contiguous()
    layer = HipMXLinear(_random_blocks(70, 4096, "e2m1", 1, dev)[0])
    for call in (lambda: mx_quantize(base), lambda: exec_fused_rmsnorm_mx(base, w), lambda: exec_fused_act_mul_mx(base, base)):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats(dev)
        had = torch.cuda.memory_allocated(dev)
        t = call()
        assert torch.cuda.max_memory_allocated(dev) - had < base.numel() * 2  # the blocks, not the values
        del t
    codes, e = H.encode(base[:1].cpu(), "e4m3")
    t = mx_quantize(base)
    assert torch.equal(H.unpack(t)[:1], codes) and torch.equal(H.scales(t)[:1], e)
    a, b = mx_quantize(part), mx_quantize(few)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    a, b = exec_fused_act_mul_mx(part, base[:, :4096]), exec_fused_act_mul_mx(few, base[:, :4096].contiguous())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    assert torch.equal(layer(part), layer(few))


def test_calls_that_are_refused(dev):
    """More rows than a call takes (here of one row's memory), inputs of no dimension."""
    from pgmoe import HipMXLinear, exec_fused_act_mul_mx, exec_fused_rmsnorm_mx, mx_quantize
    layer = HipMXLinear(_random_blocks(8, 32, "e2m1", 1, dev)[0])
    none = torch.ones((), device=dev)
    had = torch.cuda.memory_allocated(dev)
    torch.cuda.reset_peak_memory_stats(dev)
    for rows in (1 << 24, 1 << 31, (1 << 32) + 3):
        x = torch.ones(1, 32, device=dev).expand(rows, 32)
        for call in (lambda: layer(x), lambda: mx_quantize(x), lambda: exec_fused_act_mul_mx(x, x)):
            with pytest.raises(NotImplementedError, match="rows"):
                call()
    assert torch.cuda.max_memory_allocated(dev) - had < 1 << 20
    for call in (lambda: layer(none), lambda: mx_quantize(none), lambda: exec_fused_act_mul_mx(none, none),
                 lambda: exec_fused_rmsnorm_mx(none, none)):
        with pytest.raises(ValueError):
            call()


def test_layers_are_not_made_while_a_graph_is_captured(dev):
    """The refusal leaves the capture as it was: the graph holds the call before and the call behind it."""
    from pgmoe import HipMXLinear
    w, _ = _random_blocks(40, 128, "e2m1", 1, dev)
    layer = HipMXLinear(w)
    x = torch.randn(3, 128, generator=torch.Generator().manual_seed(1)).to(dev)
    want = layer(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = layer(x)
        with pytest.raises(RuntimeError, match="captured"):
            HipMXLinear(w)
        with pytest.raises(RuntimeError, match="captured"):
            HipMXLinear.from_gguf(None, "a", device=dev)
        last = layer(x)
    for _ in range(3):
        first.zero_(), last.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, want) and torch.equal(last, want) and torch.equal(layer(x), want)


def test_the_library_says_how_much_scratch_a_product_needs(dev, monkeypatch):
    """The layer asks at every call: a library that wants more gets more."""
    from pgmoe import HipMXLinear, _lib, mx
    real, asked = _lib.lib(), []

    class More:
        def __getattr__(self, name):
            return getattr(real, name)

        def pgmoe_mx_linear_values_workspace_bytes(self, rows, cols, fmt):
            asked.append((rows, cols, fmt))
            return real.pgmoe_mx_linear_values_workspace_bytes(rows, cols, fmt) + 4096

        def pgmoe_mx_linear_values(self, *a):
            assert a[-3] and a[-2] == real.pgmoe_mx_linear_values_workspace_bytes(*asked[-1]) + 4096
            return real.pgmoe_mx_linear_values(*a)

    layer = HipMXLinear(_random_blocks(70, 4128, "e2m1", 1, dev)[0], act_fmt="e2m1")
    small = HipMXLinear(_random_blocks(70, 64, "e2m1", 1, dev)[0])
    x = torch.randn(20, 4128, generator=torch.Generator().manual_seed(1)).to(dev)
    want = layer(x), layer(x[:3]), small(x[:3, :64])
    monkeypatch.setattr(mx, "lib", lambda: More())
    assert all(torch.equal(a, b) for a, b in zip((layer(x), layer(x[:3]), small(x[:3, :64])), want))
    assert asked == [(20, 4128, 4), (3, 4128, 4), (3, 64, 8)]
