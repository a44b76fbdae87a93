"""HipPagedKVCache.attend where probabilities lie far apart: keys that weigh little each and much together."""

import math

import pytest

from gpu_helpers import log
from kv_helpers import HALF_STEP

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

PAGE = 256


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda", 0)


def _heavy_and_light(dev, dt, dim, n, light, tail):
    """A cache of n keys with scores 8 (key 0) and `light` (the others), and behind them `tail` keys of -60; the
    values are 1 in column 0, 1 in column 1 but for key 0's 0, and 0 elsewhere.  The queries are the first unit vector."""
    from pgmoe import HipPagedKVCache
    pages = n // PAGE + -(-tail // PAGE)
    k = torch.zeros(pages, 1, PAGE, dim, dtype=dt, device=dev)
    v = torch.zeros_like(k)
    k[..., 0] = -60.0
    k[:n // PAGE, :, :, 0] = light
    k[0, 0, 0, 0] = 8.0
    v[..., :2] = 1.0
    v[0, 0, 0, 1] = 0.0
    return HipPagedKVCache.from_tensors(k, v)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kind", ["prompt", "decode"])
def test_light_keys_count_together(dev, kind, dim, dt):
    """One key of weight 1 and n of about 1.3 * 2^-26 each, which a run of the kernel takes together: rows enough that
    none is cut (a prompt behind a prefix, and single tokens of many sequences on the same pages).

    Tolerance: the result rounded once; each light probability rounded to fp16 after the move by 2^7, off by 2^-32
    at most (bf16: half a step of its own); the sum o takes n products in fp32, each addition off by 2^-24 of the
    sum so far, and l a sum of 16 keys a lane from every tile of 32 (32 of 64), off by 2^-24 of l; 2^-25: fp16 below its
    range."""
    from pgmoe import KVBatch
    log(f"attend light keys {kind} {dim} {dt}")
    n = 65536 if kind == "prompt" else 16384
    light = float(torch.tensor(8.0 - 26 * math.log(2.0) + math.log(1.3)).to(dt))
    w = math.exp(light - 8.0)
    if dt is torch.float16:
        assert 2.0 ** -26 < w < 2.0 ** -25
    if kind == "prompt":
        T, hq = 8192, 8
        c = _heavy_and_light(dev, dt, dim, n, light, T)
        first = n // PAGE
        b = KVBatch(torch.arange(first, first + T // PAGE, dtype=torch.int32)[None], [T], q_start=[0, T],
                    prefix_pages=torch.arange(first, dtype=torch.int32), prefix_len=n, device=dev)
    else:
        T, hq = 4096, 1
        c = _heavy_and_light(dev, dt, dim, n, light, 0)
        b = KVBatch(torch.arange(n // PAGE, dtype=torch.int32).repeat(T, 1), [n] * T, device=dev)
    q = torch.zeros(T, hq, dim, dtype=dt, device=dev)
    q[..., 0] = 1.0
    got, lse = c.attend(q, b, scale=1.0, return_lse=True)
    got, lse = got.double(), lse.double()
    total = 1.0 + (n - 1) * w
    part = (n - 1) * w / total
    half = HALF_STEP[dt]
    each = (n - 1) * (2.0 ** -32 if dt is torch.float16 else half * w)
    unit = 2.0 ** -24
    in_l = (n / 32 + 40) * unit
    for col, want in ((0, 1.0), (1, part)):
        tol = half * want + each + want * (n * unit + in_l) + 2.0 ** -25
        off = float((got[..., col] - want).abs().max())
        assert off <= tol, (col, want, off, tol)
    assert float(got[..., 2:].abs().max()) == 0.0
    assert float((lse - 8.0 - math.log(total)).abs().max()) <= in_l + 2.0 ** -20


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("dt,big,scale", [(torch.float16, 60000.0, 8.0), (torch.float16, 30000.0, 0.25), (torch.float16, 4096.0, 0.7),
                                          (torch.bfloat16, 2.0 ** 50, 1.0), (torch.bfloat16, 2.0 ** 18, 0.3)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_lens,lens,prefix", [([1, 1], [700, 33], 0), ([1], [5000], 300), ([60], [500], 0), ([100, 50], [120, 90], 400)])
def test_scores_of_any_finite_size(dev, q_lens, lens, prefix, dim, dt, big, scale, sign):
    """Scores of 10^7 to 10^30 that differ by a step of their type and more: each row is the average of the values of
    its largest scores, as the formula has it, and nothing overflows.  Ordinary queries of other rows stay as they are.

    The products of one column are exact in fp32 (11 bits by 11), scores next to each other differ by 2^-11 of `big`
    times big * scale, more than 800 units: no other key has a weight.  The average: half a step of the cache's type, V and
    the equal probabilities rounded once each."""
    from kv_helpers import Step, attend_reference
    log(f"attend far scores {q_lens} {prefix} {dim} {dt} {big} {scale} {sign}")
    s = Step(q_lens, lens, 4, 1, dim, 16, prefix, dtype=dt, seed=dim)
    k, v = s.pages()
    step = 2.0 ** -10 if dt is torch.float16 else 2.0 ** -7
    level = torch.randint(0, 9, k[..., 0].shape, generator=s.gen).double()
    kk = torch.where(torch.isnan(k), k, torch.zeros_like(k))
    kk[..., 0] = torch.where(torch.isnan(k[..., 0]), k[..., 0], (sign * big * (1 - 8 * step + level * step) * 0.5).to(dt))
    q = torch.zeros(s.T, 4, dim, dtype=dt)
    q[..., 0] = big
    q[::3, 1] = 0.0  # a row whose scores are all 0: an average of every value
    from pgmoe import HipPagedKVCache
    got, lse = HipPagedKVCache.from_tensors(kk.to(dev), v.to(dev)).attend(q.to(dev), s.batch(dev), scale=scale, return_lse=True)
    assert bool(torch.isfinite(got).all())
    out, top, _, _ = attend_reference(s, q, kk, v, scale)
    mag = v[~torch.isnan(v)].double().abs().max()
    half = HALF_STEP[dt]
    n = prefix + max(lens)
    assert float((got.double().cpu() - out).abs().max()) <= half * (2.01 * mag) + 2 * (n + 64) * 2.0 ** -24 * mag + 2.0 ** -25
    # m scale log2(e) + log2(l), times ln 2: eight roundings of 2^-24, and the sum's
    assert float(((lse.double().cpu() - top).abs() / (1 + top.abs())).max()) <= 2.0 ** -21 + (n + 64) * 2.0 ** -24
