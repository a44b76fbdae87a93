"""sample_tokens against a float64 reference (tests/kv_helpers.sample_reference): tokens equal,
log-probabilities to an fp32 step (2^-23 relative, twice the rounding of the result) and the fixed
point: weights are multiples of 2^-s with s = min(51, 62 - ceil(log2 V)) (51: what the 52-bit fraction of a
double holds), so each of V is off by 2^-(s + 1) at most, their total, 1 and more, by V 2^-(s + 1), and its
logarithm by no more."""

import math

import numpy as np
import pytest

from gpu_helpers import log
from kv_helpers import DTYPES, sample_reference

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda", 0)


def _check(dev, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    from pgmoe import sample_tokens

    def to(v, dt):
        return v.to(dev) if isinstance(v, torch.Tensor) else v

    tok, lp = sample_tokens(x.to(dev), u.to(dev), temperature=to(temperature, 0), top_k=to(top_k, 0), top_p=to(top_p, 0),
                            min_p=to(min_p, 0))
    tok, lp = tok.cpu().numpy(), lp.cpu().numpy().astype(np.float64)
    fixed = x.shape[1] * 2.0 ** -(min(51, 62 - math.ceil(math.log2(x.shape[1]))) + 1) + 2.0 ** -50
    for r in range(x.shape[0]):
        par = [float(v[r]) if isinstance(v, torch.Tensor) else v for v in (temperature, top_k, top_p, min_p)]
        par[1] = int(par[1])
        t, p = sample_reference(x[r].double().numpy(), float(u[r]), *par)
        assert tok[r] == t, (r, tok[r], t, par, float(u[r]))
        assert lp[r] == p or abs(lp[r] - p) <= 2.0 ** -23 * abs(p) + fixed, (r, lp[r], p)
    return tok


def _logits(rows, vocab, seed, dt=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * 2
    x.scatter_add_(1, torch.randint(0, vocab, (rows, min(vocab, 20)), generator=g),
                   torch.rand(rows, min(vocab, 20), generator=g) * 10)
    return x.to(dt), torch.rand(rows, generator=g)


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=1), dict(temperature=0.7, top_k=40),
            dict(top_p=0.9), dict(top_p=0.0), dict(min_p=0.05), dict(min_p=1.0), dict(temperature=3.0, top_k=500, top_p=0.7),
            dict(temperature=1.3, top_k=1000, top_p=0.99, min_p=0.001), dict(temperature=100.0, top_p=0.5),
            dict(temperature=1e-3, top_p=0.5), dict(top_k=10 ** 9), dict(temperature=50.0, top_k=3000)]


@pytest.mark.parametrize("i", range(len(SETTINGS)))
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 8192, 8193, 50001])
def test_settings_and_vocabularies(dev, vocab, i):
    log(f"sample vocab={vocab} {SETTINGS[i]}")
    for dt in ("f32", "f16", "bf16"):
        x, u = _logits(5, vocab, 100 * i + vocab % 97, DTYPES[dt])
        _check(dev, x, u, **SETTINGS[i])


@pytest.mark.parametrize("rows,vocab,dt", [(1, 151936, "f32"), (3, 262144, "bf16"), (33, 32000, "f16"), (300, 700, "f32"),
                                           (2, 1 << 20, "f16")])
def test_rows_and_large_vocabularies(dev, rows, vocab, dt):
    log(f"sample rows={rows} vocab={vocab} {dt}")
    x, u = _logits(rows, vocab, rows + vocab, DTYPES[dt])
    _check(dev, x, u, 0.8, 50, 0.95, 0.01)
    _check(dev, x, u, 1.2, 0, 0.97, 0.0)
    _check(dev, x, u, 1.0)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_ties(dev, dt):
    """Equal logits: the lower indexes are kept, at the border of each filter."""
    log(f"sample ties {dt}")
    for vocab in (10, 5000, 20000):
        x = torch.zeros(6, vocab).to(DTYPES[dt])
        u = torch.tensor([0.0, 0.1, 0.25, 0.5, 0.75, 1 - 2.0 ** -24])
        for kw in (dict(), dict(top_k=7), dict(top_p=0.5), dict(top_p=0.25, top_k=vocab // 2), dict(min_p=1.0)):
            _check(dev, x, u, **kw)
        g = torch.Generator().manual_seed(vocab)
        x = torch.randint(-3, 4, (6, vocab), generator=g).to(DTYPES[dt])  # seven values
        for kw in (dict(top_k=vocab // 3), dict(top_p=0.8), dict(top_k=11, top_p=0.5), dict(min_p=0.3), dict(top_k=1)):
            _check(dev, x, u, 0.9, **kw)
        x[:, ::2] = -0.0
        x[:, 1::2] = 0.0  # one value
        _check(dev, x, u, top_k=3)


def test_masked_and_infinite_logits(dev):
    log("sample masks")
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        x, u = _logits(9, 3001, 5, dt)
        x[0] = -math.inf                        # nothing left
        x[1] = math.nan
        x[2, 100:] = -math.inf                  # a grammar's mask
        x[3] = torch.finfo(dt).min              # the lowest value everywhere: a uniform row
        x[4, 1:] = torch.finfo(dt).min
        x[5, 7] = math.nan                      # never drawn, spoils nothing
        x[6, [5, 900, 2999]] = math.inf         # only these
        x[7, :2999] = -math.inf
        x[8] = torch.finfo(dt).max
        for kw in (dict(), dict(top_k=2), dict(top_p=0.6), dict(min_p=0.1), dict(temperature=0.0), dict(top_k=200, top_p=0.9)):
            _check(dev, x, u, **kw)


def test_every_border_of_u(dev):
    """u at 0, at the last float below 1, at 1 and past it, negative and NaN."""
    log("sample u")
    x, _ = _logits(1, 500, 8)
    for top_k in (0, 5):
        t = _check(dev, x.expand(2, -1).contiguous(), torch.tensor([0.0, 1 - 2.0 ** -24]), 0.9, top_k)
        from pgmoe import sample_tokens
        u = torch.tensor([1.0, 7.0, -1.0, math.nan], device=dev)
        got, _ = sample_tokens(x.expand(4, -1).contiguous().to(dev), u, 0.9, top_k)
        last = int(sample_reference(x[0].double().numpy(), 1.0, 0.9, top_k, 1.0, 0.0)[0])
        assert got.tolist() == [last, last, int(t[0]), int(t[0])]


def test_distribution(dev):
    """Evenly spaced u reproduce the kept distribution: each token's share is its probability to one step."""
    log("sample distribution")
    from pgmoe import sample_tokens
    n = 4096
    x, _ = _logits(1, 50, 3)
    u = (torch.arange(n, dtype=torch.float32) + 0.5) / n
    tok, lp = sample_tokens(x.expand(n, -1).to(dev), u.to(dev), 1.5, 20)
    cnt = np.bincount(tok.cpu().numpy(), minlength=50)
    for t in np.nonzero(cnt)[0]:
        p = math.exp(float(lp[(tok == int(t))][0]))
        assert abs(cnt[t] - p * n) <= 1.0 + 1e-3
    assert (cnt > 0).sum() <= 20


def test_parameters_by_row(dev):
    log("sample rows' own parameters")
    x, u = _logits(40, 4000, 21, torch.float16)
    g = torch.Generator().manual_seed(2)
    temp = torch.rand(40, generator=g) * 2
    temp[::5] = 0.0
    k = torch.randint(0, 300, (40,), generator=g, dtype=torch.int32)
    k[3], k[4] = -1, 4000
    p = torch.rand(40, generator=g)
    p[::3] = 1.0
    m = torch.rand(40, generator=g) * 0.1
    m[::2] = 0.0
    _check(dev, x, u, temp, k, p, m)
    _check(dev, x, u, temp, 10, p, 0.0)


def test_layouts_graphs_and_refusals(dev):
    from pgmoe import sample_tokens
    log("sample layouts")
    x, u = _logits(6, 1000, 4)
    wide = torch.full((6, 1300), 99.0)
    wide[:, 100:1100] = x
    want = sample_tokens(x.to(dev), u.to(dev), 0.8, 30, 0.9)
    g = wide.to(dev)
    for view in (g[:, 100:1100], g[:, 100:1100].t().contiguous().t()):
        got = sample_tokens(view, u.to(dev), 0.8, 30, 0.9)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    half = x.half().to(dev)
    odd = torch.empty(6 * 1000 + 1, dtype=torch.float16, device=dev)[1:].view(6, 1000)  # 2-byte aligned rows
    odd.copy_(half)
    a, b = sample_tokens(half, u.to(dev), 0.8, 30, 0.9), sample_tokens(odd, u.to(dev), 0.8, 30, 0.9)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    xs, us = x.to(dev), u.to(dev)
    with torch.cuda.stream(s):
        sample_tokens(xs, us, 0.8, 30, 0.9)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            out = sample_tokens(xs, us, 0.8, 30, 0.9)
    for seed in range(4):
        x2, u2 = _logits(6, 1000, 50 + seed)
        xs.copy_(x2)
        us.copy_(u2)
        w = sample_tokens(xs, us, 0.8, 30, 0.9)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])
    del gr
    x, u = x.to(dev), u.to(dev)
    for kw in (dict(temperature=-1.0), dict(top_p=float("nan")), dict(min_p=-0.1), dict(top_k=torch.ones(6, device=dev)),
               dict(temperature=torch.ones(5, device=dev))):
        with pytest.raises(ValueError):
            sample_tokens(x, u, **kw)
    with pytest.raises(NotImplementedError):
        sample_tokens(x.double(), u)
    with pytest.raises(ValueError):
        sample_tokens(x, u[:5])
    with pytest.raises(ValueError):
        sample_tokens(x, u.double())
    assert sample_tokens(x[:0], u[:0])[0].shape == (0,)


def test_borders_far_from_the_maximum(dev):
    """The last kept token lies so far below the maximum that its weight is some units of the fixed point, or
    none: 200 logits 0.4 apart, and one row of a large vocabulary at a low temperature.

    u = 0 draws the first token that has a weight: one of half a unit, 2^-52 for 200 tokens, at least.  (Weights
    0.4 apart in logarithm: the nearest to 2^-52 = e^-36.04 is e^-36, 4 % above, far from the 2^-50 that the
    kernel's are off by.  Together the tokens without weight have at most 200 * 2^-52 of the probability, and u
    in (0, 2^-24) is not drawn by any generator of 24 bits.)"""
    from pgmoe import sample_tokens
    log("sample far borders")
    g = torch.Generator().manual_seed(12)
    place = torch.randperm(200, generator=g)
    x = (-0.4 * torch.arange(200.0))[place].expand(6, -1).contiguous()
    u = torch.tensor([0.0, 0.2, 0.5, 0.9, 0.99, 1 - 2.0 ** -24])
    for top_k in (77, 79, 80, 81, 90, 150, 199):
        for min_p, least in ((0.0, 2.0 ** -52), (1e-15, 1e-15)):
            _check(dev, x[1:], u[1:], 1.0, top_k, 1.0, min_p)
            tok, _ = sample_tokens(x[:1].to(dev), u[:1].to(dev), 1.0, top_k, 1.0, min_p)
            drawn = (place < top_k) & (torch.exp(x[0].double()) >= least)
            assert int(tok) == int(drawn.nonzero()[0])
    for vocab in (9000, 131072):
        x, u = _logits(3, vocab, 31)
        _check(dev, x, u, 0.02, 2000)
        _check(dev, x, u, 0.05, vocab - 5, 0.999)


def test_more_rows_than_a_grid_axis(dev):
    """70000 rows: the same tokens as in two calls of half as many."""
    log("sample many rows")
    from pgmoe import sample_tokens
    x, u = _logits(70000, 5, 77)
    x, u = x.to(dev), u.to(dev)
    tok, lp = sample_tokens(x, u, 0.9, 3, 0.9)
    for a in (0, 35000):
        t, p = sample_tokens(x[a:a + 35000], u[a:a + 35000], 0.9, 3, 0.9)
        assert torch.equal(tok[a:a + 35000], t) and torch.equal(lp[a:a + 35000], p)
    _check(dev, x[69990:].cpu(), u[69990:].cpu(), 0.9, 3, 0.9)


def test_two_streams_at_once(dev):
    log("sample two streams")
    from pgmoe import sample_tokens
    a, b = [(x.to(dev), u.to(dev)) for x, u in (_logits(40, 60000, 1), _logits(7, 131072, 2, torch.float16))]
    kw = dict(temperature=0.9, top_k=300, top_p=0.95)
    want = [sample_tokens(*a, **kw), sample_tokens(*b, **kw)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for _ in range(8):
        for st, x in zip(streams, (a, b)):
            with torch.cuda.stream(st):
                outs.append(sample_tokens(*x, **kw))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o[0], want[i % 2][0]) and torch.equal(o[1], want[i % 2][1]), i
