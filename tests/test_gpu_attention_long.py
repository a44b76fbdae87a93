"""HipPagedKVCache.attend on calls large enough for every way the work is dealt: row tiles past what a lane sums by
itself (16) and past what a wave looks through at a time (64), hundreds of sequences that each fill shared row
tiles, and prompts beside long decodes, where a row has few partial slots and runs get long.

float64 on the device for sequences or tokens of the call (all of them where that is quick), with the tolerance of
kv_helpers.attend_reference; every other row has to be written and finite.  Unused rows of pages hold NaN."""

import math

import pytest

from gpu_helpers import log
from kv_helpers import DTYPES, HALF_STEP, Step

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda", 0)


def _pages(s, dev):
    """As Step.pages, on the device."""
    g = torch.Generator(dev).manual_seed(s.seed + 1)
    shape = (s.n_pages, s.hkv, s.page, s.dim)
    used = torch.zeros(s.n_pages, s.page, dtype=torch.bool)

    def mark(pages, n):
        full, rest = divmod(n, s.page)
        used[pages[:full].long()] = True
        if rest:
            used[int(pages[full]), :rest] = True

    mark(s.prefix_pages, s.prefix)
    for b, n in enumerate(s.lens):
        mark(s.table[b], n)
    dead = ~used.to(dev)[:, None, :, None]
    return [torch.randn(shape, generator=g, device=dev).to(s.dtype).masked_fill_(dead, math.nan) for _ in range(2)]


def _rows(s, cache, b, head):
    """The prefix's rows and sequence b's own ones, float64 [prefix + lens[b], dim]."""
    def some(pages, n):
        return cache[pages[:-(-n // s.page)].long().to(cache.device), head].reshape(-1, s.dim)[:n]

    return torch.cat((some(s.prefix_pages, s.prefix), some(s.table[b], s.lens[b]))).double()


def _check(dev, s, sequences=None, tokens=None):
    """Runs the call; `sequences` of it (None: all), of each at most `tokens` tokens spread over it and its last."""
    from pgmoe import HipPagedKVCache
    k, v = _pages(s, dev)
    q = torch.randn(s.T, s.hq, s.dim, generator=torch.Generator(dev).manual_seed(s.seed), device=dev).to(s.dtype)
    out = torch.full((s.T, s.hq, s.dim), 777.0, dtype=s.dtype, device=dev)
    cache = HipPagedKVCache.from_tensors(k, v)
    got, lse = cache.attend(q, s.batch(dev), out=out, return_lse=True)
    n = s.q_start[-1]
    assert bool(torch.isfinite(got).all()) and bool(((got == 777.0).all(-1) == (torch.arange(s.T, device=dev) >= n)[:, None]).all())
    g, half, unit, scale = s.hq // s.hkv, HALF_STEP[s.dtype], 2.0 ** -24, s.dim ** -0.5
    for b in range(len(s.lens)) if sequences is None else sequences:
        m, ln = s.q_lens[b], s.lens[b]
        if not m:
            continue
        pick = torch.arange(m) if tokens is None or m <= tokens else torch.linspace(0, m - 1, tokens).round().long().unique()
        see = (s.prefix + ln - m + 1 + pick).to(dev)
        late = torch.arange(s.prefix + ln, device=dev)[None, :] >= see[:, None]
        at = (s.q_start[b] + pick).to(dev)
        for h in range(s.hkv):
            kk, vv = _rows(s, k, b, h), _rows(s, v, b, h)
            for i in range(h * g, (h + 1) * g):
                qq = q[at, i].double()
                x = (qq @ kk.T * scale).masked_fill(late, -math.inf)
                w = torch.softmax(x, -1)
                o, a = w @ vv, w @ vv.abs()
                mag = (qq.abs() @ kk.abs().T * scale).masked_fill(late, 0).amax(-1, keepdim=True)
                ds = unit * ((s.dim + 4) * mag + 3 * x.masked_fill(late, 0).abs().amax(-1, keepdim=True))
                terms = (see[:, None] + 64) * unit
                tol = half * o.abs() + a * (1.01 * half + 2 * ds + 2 * terms) + 2.0 ** -25
                d = (got[at, i].double() - o).abs()
                assert bool((d <= tol).all()), (b, i, float((d - tol).max()))
                ll = torch.logsumexp(x, -1, keepdim=True)
                ld = (lse[at, i, None].double() - ll).abs()
                assert bool((ld <= ds + terms + 4 * unit * ll.abs()).all()), (b, i, float(ld.max()))


@pytest.mark.parametrize("dim,dt", [(64, "bf16"), (128, "f16"), (256, "bf16")])
@pytest.mark.parametrize("tokens,before,prefix", [(300, 0, 0), (300, 57, 211), (1100, 0, 0), (1100, 301, 1033)])
def test_one_long_prompt(dev, tokens, before, prefix, dim, dt):
    """19 and 69 row tiles a KV head."""
    log(f"attend prompt of {tokens} behind {prefix} + {before}, dim {dim}")
    s = Step([tokens], [tokens + before], 16, 2, dim, 32, prefix, extra=2, dtype=DTYPES[dt], seed=tokens + prefix)
    _check(dev, s, tokens=None if dim == 64 else 150)


@pytest.mark.parametrize("prefix", [0, 333])
@pytest.mark.parametrize("long", [0, 300])
def test_hundreds_of_sequences_with_row_tiles_of_their_own(dev, long, prefix):
    """300 sequences of 5 to 9 tokens, 40 to 72 rows a KV head, two sequences a thread; one of them a prompt."""
    log(f"attend 300 shared sequences, long {long}, prefix {prefix}")
    q = [5 + i % 5 for i in range(300)]
    lens = [n + (i * 37) % 290 for i, n in enumerate(q)]
    if long:
        q[211], lens[211] = long, long + 50
    s = Step(q, lens, 8, 1, 64, 16, prefix, dtype=torch.float16, seed=4)
    _check(dev, s)
    # with single tokens, and sequences without a token, between them
    q = [(0, 1, 6, 1, 9)[i % 5] for i in range(300)]
    lens = [n + (i * 53) % 400 for i, n in enumerate(q)]
    s = Step(q, lens, 16, 2, 128, 64, prefix, dtype=torch.bfloat16, seed=5)
    _check(dev, s)


def test_the_most_sequences_with_several_tokens(dev):
    """4096 sequences, 16 a thread, of 0, 1 and 5 tokens at 8 query heads on one: both kinds of segment."""
    log("attend 4096 sequences of several tokens")
    q = [(0, 1, 5, 5, 1, 0, 5)[i % 7] for i in range(4096)]
    lens = [n + (i * 11) % 70 for i, n in enumerate(q)]
    s = Step(q, lens, 8, 1, 64, 16, 50, dtype=torch.float16, seed=6)
    _check(dev, s, sequences=range(0, 4096, 23))


@pytest.mark.parametrize("prompts,decodes,hq,hkv,dim,prefix,dt", [
    ([2048, 300], [30011, 17], 32, 8, 128, 0, "f16"),       # 6 slots a row
    ([2048, 300], [30011, 17], 32, 8, 128, 1000, "bf16"),
    ([4096], [20000] + [40] * 30, 32, 4, 128, 0, "bf16"),   # 4 slots, the least
    ([1500, 1000], [12000, 9000, 5], 16, 2, 256, 70, "f16"),
    ([4096, 4100], [25000], 64, 8, 64, 500, "f16"),
])
def test_prompts_beside_long_decodes(dev, prompts, decodes, hq, hkv, dim, prefix, dt):
    """A server's mixed step: many rows leave few partial slots a row, and the long single-token sequences are cut into
    that many pieces at most."""
    log(f"attend prompts {prompts} beside decodes {decodes[:3]} dim {dim} prefix {prefix}")
    q = prompts + [1] * len(decodes)
    s = Step(q, [n + 33 for n in prompts] + decodes, hq, hkv, dim, 64, prefix, dtype=DTYPES[dt], seed=dim + prefix)
    _check(dev, s, tokens=40)


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("prefix", [0, 4000])
def test_many_single_tokens_in_parts(dev, dim, prefix):
    """More than 2048 rows whose partial rows one group of threads each merges."""
    log(f"attend 150 long decodes, dim {dim}, prefix {prefix}")
    s = Step([1] * 150, [700 + (i * 131) % 2500 for i in range(150)], 32, 2, dim, 64, prefix, dtype=torch.float16, seed=dim)
    _check(dev, s, sequences=range(0, 150, 7))
