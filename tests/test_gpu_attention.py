"""HipPagedKVCache.append / .attend against float64 references (tests/kv_helpers.py).

Every unused row of every page holds NaN, page-table entries past a sequence's pages hold -1, so that
a read of what is masked shows in the result.  Tolerances are derived in kv_helpers from the roundings
the entry points document."""

import math

import pytest

from gpu_helpers import log
from kv_helpers import DTYPES, HALF_STEP, Step, attend_reference, check_attend, norm_reference, rotate_reference

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda", 0)


def _cache(dev, k, v):
    from pgmoe import HipPagedKVCache
    return HipPagedKVCache.from_tensors(k.to(dev), v.to(dev))


def _run(dev, s, scale=None, qscale=1.0):
    k, v = s.pages()
    q = s.q(qscale)
    out = torch.full((s.T, s.hq, s.dim), 7.0, dtype=s.dtype, device=dev)
    got, lse = _cache(dev, k, v).attend(q.to(dev), s.batch(dev), scale=scale, out=out, return_lse=True)
    torch.cuda.synchronize()
    assert got.data_ptr() == out.data_ptr()
    ref = attend_reference(s, q, k, v, scale)
    check_attend(s, got, ref, lse)
    assert bool((got[s.q_start[-1]:] == 7.0).all()), "rows behind the last sequence were written"
    return got, lse


# ------------------------------------------------------------------ attend
SHAPES = [
    # q_lens, lens, hq, hkv, dim, page, prefix, dtype
    ([1], [1], 1, 1, 64, 16, 0, "f16"),
    ([1], [0], 4, 2, 128, 16, 0, "f16"),                        # no key at all
    ([1], [0], 4, 2, 128, 16, 1, "bf16"),                       # one shared key
    ([1] * 3, [5, 0, 33], 8, 2, 64, 16, 0, "bf16"),             # an empty sequence between others
    ([1] * 4, [31, 32, 33, 64], 8, 1, 128, 32, 0, "f16"),       # around a tile
    ([1] * 3, [1, 40, 257], 16, 2, 128, 16, 100, "f16"),        # a prefix that ends inside a page
    ([1] * 3, [15, 16, 17], 7, 7, 256, 16, 63, "bf16"),         # one head a KV head
    ([1] * 2, [700, 3], 10, 2, 256, 128, 129, "f16"),           # 5 : 1 heads
    ([1] * 9, [64] * 9, 32, 4, 128, 64, 512, "bf16"),           # whole pages throughout
    ([1] * 40, list(range(40)), 8, 4, 64, 16, 200, "f16"),
    ([1] * 70, [(37 * i) % 90 for i in range(70)], 16, 2, 128, 16, 333, "bf16"),  # many rows on the prefix
    ([1], [2500], 32, 8, 128, 16, 0, "f16"),                    # a long axis for few rows
    ([1] * 2, [1, 2000], 8, 1, 64, 64, 1500, "bf16"),
    ([3, 1, 5], [10, 70, 5], 8, 2, 128, 16, 40, "f16"),         # draft tokens
    ([4, 0, 2], [4, 50, 90], 16, 1, 128, 32, 0, "bf16"),        # a sequence without a token
    ([8] * 5, [8, 9, 40, 41, 200], 32, 4, 64, 16, 77, "f16"),
    ([70, 1, 33], [70, 300, 200], 8, 4, 128, 16, 0, "bf16"),    # prompts beside a decode
    ([150], [150], 4, 4, 128, 64, 130, "f16"),
    ([40, 200], [45, 500], 8, 1, 64, 32, 65, "f16"),
    ([90], [260], 6, 2, 256, 16, 17, "bf16"),
    ([3, 2], [1, 2], 4, 2, 128, 16, 0, "f16"),                  # more queries than keys: rows that see nothing
    ([5], [2], 4, 2, 64, 16, 20, "bf16"),                       # the same behind a prefix
]


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_attend_matches_float64(dev, i):
    q_lens, lens, hq, hkv, dim, page, prefix, dt = SHAPES[i]
    log(f"attend {SHAPES[i][2:]} q={q_lens[:6]} lens={lens[:6]}")
    s = Step(q_lens, lens, hq, hkv, dim, page, prefix, dtype=DTYPES[dt], seed=i, extra=0)
    _run(dev, s)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("q_lens,lens,prefix", [([1, 1, 1], [20, 0, 7], 50), ([3, 40], [9, 60], 0)])
def test_rows_behind_the_last_sequence_are_left(dev, q_lens, lens, prefix, dt):
    log(f"attend extra rows {q_lens} {dt}")
    _run(dev, Step(q_lens, lens, 8, 2, 128, 16, prefix, extra=5, dtype=DTYPES[dt], seed=3))


@pytest.mark.parametrize("qscale,scale", [(30.0, None), (1.0, 2.0), (0.01, None), (8.0, 0.001)])
def test_attend_scales(dev, qscale, scale):
    """Scores in the hundreds (a softmax of one key) and near zero (an average)."""
    log(f"attend qscale={qscale} scale={scale}")
    _run(dev, Step([1, 2], [300, 80], 8, 2, 128, 16, 100, dtype=torch.float16, seed=5), scale, qscale)


def test_lowest_values_and_infinities(dev):
    """Keys that give -inf scores get no weight; a row whose every score is -inf is NaN as softmax has it;
    a +inf in V shows in the rows that see it and in no other."""
    log("attend infinities")
    s = Step([1, 1, 3], [40, 8, 35], 4, 1, 128, 16, 0, dtype=torch.float16, seed=9)
    k, v = s.pages()
    q = s.q().abs() + 0.1
    low = torch.finfo(torch.float16).min

    def row(b, j):
        return int(s.table[b, j // 16]), 0, j % 16

    k[row(0, 3)] = -math.inf
    k[row(0, 20)] = low
    for j in range(8):
        k[row(1, j)] = -math.inf
    v[row(2, 34)] = math.inf  # the last key: only the last of the three queries sees it
    v[row(2, 33)][5] = math.nan  # seen by the last two
    got = _cache(dev, k, v).attend(q.to(dev), s.batch(dev)).cpu().double()
    ok0 = [j for j in range(40) if j != 3]
    x = q[0].double() @ s.keys(0, 40, k, 0)[ok0].T / math.sqrt(128)
    o = torch.softmax(x, -1) @ s.keys(0, 40, v, 0)[ok0]
    assert bool(((got[0] - o).abs() <= 2.0 ** -9 * (o.abs() + 2)).all())
    assert bool(torch.isnan(got[1]).all())
    assert bool(torch.isfinite(got[2]).all())
    assert bool(torch.isnan(got[3][:, 5]).all()) and bool(torch.isfinite(got[3][:, :5]).all())
    assert not bool(torch.isfinite(got[4]).any())
    x = q[2].double() @ s.keys(2, 33, k, 0).T / math.sqrt(128)
    o = torch.softmax(x, -1) @ s.keys(2, 33, v, 0)
    assert bool(((got[2] - o).abs() <= 2.0 ** -9 * (o.abs() + 2)).all())


def test_a_row_that_is_not_finite_leaves_the_others(dev):
    """NaN queries of one token change no bit of the others', decode and prompt rows, prefix and own keys."""
    log("attend NaN query")
    s = Step([1, 40, 1], [30, 90, 200], 8, 2, 128, 16, 70, dtype=torch.bfloat16, seed=2)
    k, v = s.pages()
    q = s.q().to(dev)
    c, b = _cache(dev, k, v), s.batch(dev)
    a = c.attend(q, b).clone()
    q2 = q.clone()
    q2[5] = math.nan
    d = c.attend(q2, b)
    keep = [t for t in range(s.T) if t != 5]
    assert torch.equal(a[keep], d[keep]) and bool(torch.isnan(d[5]).all())


def test_pages_that_do_not_exist(dev):
    """A key on a page outside the cache, or past the page table, gives NaN to the rows that see it."""
    log("attend bad pages")
    s = Step([1, 1, 1, 2], [60, 60, 60, 33], 8, 2, 128, 16, 40, dtype=torch.float16, seed=4)
    k, v = s.pages()
    q = s.q()
    ref = attend_reference(s, q, k, v)
    batch = s.batch(dev)
    batch.page_table[1, 2] = -1
    batch.page_table[2, 0] = s.n_pages
    batch.page_table[3, 2] = 2 ** 31 - 1  # own key 32: the second query's own
    got = _cache(dev, k, v).attend(q.to(dev), batch).cpu().double()
    assert bool(((got[0] - ref[0][0]).abs() <= ref[2][0]).all())
    assert bool(torch.isnan(got[1]).all()) and bool(torch.isnan(got[2]).all())
    assert bool(((got[3] - ref[0][3]).abs() <= ref[2][3]).all())
    assert bool(torch.isnan(got[4]).all())
    batch = s.batch(dev)
    batch.lens[0] = 1000  # past the table
    batch.lens[1] = 2 ** 31 - 1
    batch.lens[2] = -5
    got = _cache(dev, k, v).attend(q.to(dev), batch).cpu().double()
    assert bool(torch.isnan(got[0]).all()) and bool(torch.isnan(got[1]).all())
    assert bool(torch.isfinite(got[2]).all())  # a negative length: the prefix alone
    batch = s.batch(dev)
    batch.prefix_pages[1] = -7
    assert bool(torch.isnan(_cache(dev, k, v).attend(q.to(dev), batch)).all())


def test_q_start_that_is_out_of_range_stays_inside(dev):
    """Rows beyond the call's tokens are not written, whatever q_start holds."""
    log("attend q_start out of range")
    from pgmoe import KVBatch
    s = Step([2, 3], [20, 30], 8, 2, 128, 16, 10, dtype=torch.float16, seed=6)
    k, v = s.pages()
    buf = torch.full((s.T + 8, 8, 128), 3.0, dtype=torch.float16, device=dev)
    b = KVBatch(s.table.to(dev), torch.tensor(s.lens, dtype=torch.int32, device=dev),
                q_start=torch.tensor([0, 2, 400], dtype=torch.int32, device=dev), prefix_pages=s.prefix_pages.to(dev),
                prefix_len=10)
    _cache(dev, k, v).attend(s.q().to(dev), b, out=buf[:s.T])
    assert bool((buf[s.T:] == 3.0).all())


@pytest.mark.parametrize("layout", ["layer_slice", "interleaved", "token_major"])
def test_strided_caches_and_queries(dev, layout):
    """Pages inside a larger allocation, and queries that are a part of a fused projection."""
    log(f"attend layout {layout}")
    s = Step([1, 4, 1], [50, 60, 0], 8, 2, 128, 16, 30, dtype=torch.bfloat16, seed=8)
    k, v = s.pages()
    n = s.n_pages
    if layout == "layer_slice":
        big = torch.full((2, n, 3, 2, 16, 128), math.nan, dtype=s.dtype, device=dev)
        kk, vv = big[0, :, 1], big[1, :, 1]
    elif layout == "interleaved":
        big = torch.full((n, 2, 2, 16, 128), math.nan, dtype=s.dtype, device=dev)
        kk, vv = big[:, 0], big[:, 1]
    else:
        big = torch.full((2, n, 16, 2, 128), math.nan, dtype=s.dtype, device=dev)
        kk, vv = big[0].transpose(1, 2), big[1].transpose(1, 2)
    kk.copy_(k)
    vv.copy_(v)
    from pgmoe import HipPagedKVCache
    cat = s.randn(s.T, 12 * 128).to(s.dtype)
    q = cat[:, :8 * 128].unflatten(1, (8, 128))
    c = HipPagedKVCache.from_tensors(kk, vv)
    ref = attend_reference(s, q, k, v)
    check_attend(s, c.attend(cat.to(dev)[:, :8 * 128].unflatten(1, (8, 128)), s.batch(dev)), ref)
    odd = torch.empty(s.T * 8 * 128 + 1, dtype=s.dtype, device=dev)[1:].view(s.T, 8, 128)  # not 16-byte aligned
    odd.copy_(q)
    check_attend(s, c.attend(odd, s.batch(dev)), ref)


def test_offsets_past_32_bits(dev):
    """Pages whose byte and element offsets pass 2^32."""
    log("attend + append far pages")
    from pgmoe import HipPagedKVCache, KVBatch
    n = (1 << 32) // (1 * 16 * 128) // 8 + 64  # strided eightfold: 2^32 elements and some
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GiB of free GPU memory")
    big = torch.empty(2, n, 8, 16, 128, dtype=torch.float16, device=dev)
    c = HipPagedKVCache.from_tensors(big[0, :, :1], big[1, :, :1])
    table = torch.tensor([[n - 1, 0, n - 2]], dtype=torch.int32, device=dev)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(40, 1, 128, generator=g).to(torch.float16) for _ in range(2))
    q = torch.randn(40, 4, 128, generator=g).to(torch.float16)
    b = KVBatch(table, [40], q_start=[0, 40])
    qr = c.append(q.to(dev), k.to(dev), v.to(dev), b)
    assert torch.equal(qr.cpu(), q) and torch.equal(big[0, n - 1, 0].cpu(), k[:16, 0])
    assert torch.equal(big[1, n - 2, 0, :8].cpu(), v[32:, 0])
    x = torch.einsum("qhd,kd->hqk", q.double(), k[:, 0].double()) / math.sqrt(128)
    x = x.masked_fill(torch.ones(40, 40).triu(1).bool(), -math.inf)
    o = torch.einsum("hqk,kd->qhd", torch.softmax(x, -1), v[:, 0].double())
    assert bool(((c.attend(qr, b).cpu().double() - o).abs() <= 2.0 ** -9 * (o.abs() + 2)).all())
    del big, c
    torch.cuda.empty_cache()


def test_attend_refusals(dev):
    from pgmoe import HipPagedKVCache, KVBatch
    c = HipPagedKVCache(8, 16, 2, 128, device=dev)
    table = torch.zeros(2, 3, dtype=torch.int32, device=dev)
    b = KVBatch(table, [4, 5])
    q = torch.zeros(2, 4, 128, dtype=torch.float16, device=dev)
    with pytest.raises(ValueError, match="q_start"):
        c.attend(torch.zeros(3, 4, 128, dtype=torch.float16, device=dev), b)
    with pytest.raises(ValueError, match="query heads"):
        c.attend(torch.zeros(2, 3, 128, dtype=torch.float16, device=dev), b)
    with pytest.raises(NotImplementedError, match="dtype"):
        c.attend(q.float(), b)
    with pytest.raises(ValueError):
        c.attend(q[..., :64], b)
    with pytest.raises(ValueError, match="overlaps"):
        c.attend(q, b, out=q)
    with pytest.raises(ValueError, match="scale"):
        c.attend(q, b, scale=0.0)
    with pytest.raises(ValueError, match="cuda|cache"):
        c.attend(q.cpu(), b)
    with pytest.raises(ValueError, match="prefix"):
        c.attend(q, KVBatch(table, [4, 5], prefix_pages=[1, 2], prefix_len=33))
    for bad in ([0, 2, 1], [1, 2, 3]):
        with pytest.raises(ValueError, match="q_start"):
            KVBatch(table, [4, 5], q_start=bad)
    with pytest.raises(ValueError, match="q_start"):
        KVBatch(table, [4, 5], q_start=[0, 2])
    with pytest.raises(ValueError, match="lens"):
        KVBatch(table, [4, -5])
    with pytest.raises(ValueError, match="int32"):
        KVBatch(table.long(), [4, 5])
    with pytest.raises(NotImplementedError, match="sequences"):
        KVBatch(torch.zeros(4097, 1, dtype=torch.int32, device=dev), [1] * 4097)
    k = torch.zeros(8, 2, 16, 136, dtype=torch.float16, device=dev)
    with pytest.raises(ValueError):
        HipPagedKVCache.from_tensors(k[..., 4:132], k[..., 4:132])  # rows not 16-byte aligned
    with pytest.raises(ValueError, match="overlap"):
        HipPagedKVCache.from_tensors(k[:1, ..., :128].expand(8, 2, 16, 128), k[:1, ..., :128].expand(8, 2, 16, 128))
    assert c.attend(torch.zeros(0, 4, 128, dtype=torch.float16, device=dev), KVBatch(table, [4, 5], q_start=[0, 0, 0])).shape == (0, 4, 128)


def test_many_sequences(dev):
    """4096 sequences (the most a batch takes), one in 200 of them with keys of its own."""
    log("attend 4096 sequences")
    n = 4096
    s = Step([1] * n, [(i % 7) * (i % 200 == 0) for i in range(n)], 2, 1, 64, 16, 3, dtype=torch.float16, seed=1)
    _run(dev, s)
    s = Step([int(i % 3 == 0) for i in range(n)], [(i % 5) * (i % 100 == 0) for i in range(n)], 2, 1, 64, 16, 2,
             extra=3, dtype=torch.float16, seed=1)
    _run(dev, s)


def test_graphs_and_streams(dev):
    """Two captured decode steps of different batches replayed in turn and side by side, with eager calls
    between, on lengths that advance in place; every replay against an eager call."""
    log("attend graphs")
    steps = [Step([1] * 6, [40, 41, 100, 3, 17, 64], 8, 2, 128, 16, 150, dtype=torch.float16, seed=11),
             Step([3, 50], [20, 300], 16, 2, 128, 32, 0, dtype=torch.float16, seed=12)]
    made = []
    for s in steps:
        k, v = s.pages(poison=0.25)  # lengths grow into rows that hold a value
        made.append((_cache(dev, k, v), s.q().to(dev), s.batch(dev)))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(st):
        for c, q, b in made:
            c.attend(q, b)
        torch.cuda.synchronize()
        for c, q, b in made:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                outs.append(c.attend(q, b, return_lse=True))
            graphs.append(g)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for rep in range(4):
        want = [c.attend(q, b, return_lse=True) for c, q, b in made]
        torch.cuda.synchronize()
        for o in outs:
            o[0].fill_(-1.0)
            o[1].fill_(-1.0)
        torch.cuda.synchronize()
        if rep % 2:
            with torch.cuda.stream(st):
                graphs[0].replay()
            with torch.cuda.stream(other):
                graphs[1].replay()
        else:
            for g in graphs:
                g.replay()
            made[0][0].attend(made[0][1], made[0][2])
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            assert torch.equal(w[0], o[0]) and torch.equal(w[1], o[1]), rep
        for (_, _, b), s in zip(made, steps):
            b.lens.copy_(torch.tensor([min(n + 5 * (rep + 1), s.table.shape[1] * s.page, ((n - 1) // s.page + 1) * s.page)
                                       for n in s.lens], dtype=torch.int32))
    del graphs


def test_repeats_are_the_same_bits(dev):
    log("attend repeats")
    s = Step([1] * 20, [(91 * i) % 700 for i in range(20)], 16, 2, 128, 16, 1000, dtype=torch.bfloat16, seed=13)
    k, v = s.pages()
    c, q, b = _cache(dev, k, v), s.q().to(dev), s.batch(dev)
    a, la = c.attend(q, b, return_lse=True)
    for _ in range(5):
        o, lo = c.attend(q, b, return_lse=True)
        assert torch.equal(a, o) and torch.equal(la, lo)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_lens,lens,prefix", [([1, 1], [700, 90], 0), ([2, 1], [300, 40], 700), ([70], [400], 0),
                                                ([40] * 4, [60, 50, 40, 45], 600)])
def test_scores_that_grow_along_the_keys(dev, dim, q_lens, lens, prefix):
    """Every key's scores are larger than those before it, by up to 60 in all: the running maximum moves
    throughout, and the sums are rescaled."""
    log(f"attend growing scores dim={dim} q={q_lens} prefix={prefix}")
    s = Step(q_lens, lens, 8, 2, dim, 16, prefix, dtype=torch.float16, seed=dim + prefix)
    k, v = s.pages()
    c = 60.0 / (0.64 * dim ** 0.5)
    for j in range(prefix):
        at = int(s.prefix_pages[j // 16]), slice(None), j % 16
        k[at] = (k[at].float().abs() * (c * j / (prefix + max(lens)))).half()
    for b, n in enumerate(lens):
        for j in range(n):
            at = int(s.table[b, j // 16]), slice(None), j % 16
            k[at] = (k[at].float().abs() * (c * (prefix + j) / (prefix + max(lens)))).half()
    q = s.q().abs()
    got, lse = _cache(dev, k, v).attend(q.to(dev), s.batch(dev), return_lse=True)
    check_attend(s, got, attend_reference(s, q, k, v), lse)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,prefix", [(1, 0), (1, 40), (6, 0), (60, 0), (60, 40), (200, 17)])
def test_values_that_are_not_finite(dev, dim, n, prefix):
    """Infinite and NaN values of keys that some or all queries see show in their column of the rows that see
    them; every other value is as if they were not there."""
    log(f"attend bad values dim={dim} n={n} prefix={prefix}")
    ln = n + 37
    s = Step([n], [ln], 4, 1, dim, 16, prefix, dtype=torch.bfloat16, seed=n + dim)
    k, v = s.pages()
    q = s.q()
    clean = v.clone()
    seen = torch.zeros(n, dim, dtype=torch.bool)
    for j, col, x in ((ln - 1, 3, math.inf), (ln - 2, 7, math.nan), (5, 11, -math.inf), (ln - 1 - n // 2, 60, math.nan)):
        at = int(s.table[0, j // 16]), 0, j % 16, col
        clean[at], v[at] = 0, x
        seen[max(0, j - (ln - n)):, col] = True
    out, _, tol, _ = attend_reference(s, q, k, clean)
    got = _cache(dev, k, v).attend(q.to(dev), s.batch(dev)).cpu().double()
    bad = seen[:, None].expand(n, 4, dim)
    assert not bool(torch.isfinite(got[bad]).any())
    assert bool(((got - out).abs() <= tol)[~bad].all())


def test_two_streams_at_once(dev):
    """Calls on two streams side by side, 256-wide heads and 128-wide ones: the bits of calls one by one."""
    log("attend two streams")
    made = []
    for dim, seed in ((256, 3), (128, 4)):
        s = Step([1] * 12 + [50], [(67 * i) % 500 for i in range(12)] + [300], 8, 2, dim, 16, 300, dtype=torch.bfloat16, seed=seed)
        k, v = s.pages()
        made.append((_cache(dev, k, v), s.q().to(dev), s.batch(dev)))
    want = [c.attend(q, b) for c, q, b in made]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for _ in range(8):
        for st, (c, q, b) in zip(streams, made):
            with torch.cuda.stream(st):
                outs.append(c.attend(q, b))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, want[i % 2]), i


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("dim,rot,inter,hq,hkv,norm", [(128, 128, False, 8, 2, True), (128, 64, True, 5, 5, False),
                                                       (64, 64, False, 4, 1, True), (256, 96, False, 3, 1, False),
                                                       (256, 256, True, 8, 4, True), (64, 16, False, 16, 2, False),
                                                       (128, 0, False, 4, 2, True)])
def test_append_matches_float64(dev, src, dt, dim, rot, inter, hq, hkv, norm):
    log(f"append dim={dim} rot={rot} inter={inter} {src}->{dt}")
    from pgmoe import HipRotary
    s = Step([1, 20, 3, 0], [1000, 20, 40, 9], hq, hkv, dim, 16, 37, extra=3, dtype=DTYPES[dt], seed=dim + rot)
    k0, v0 = s.pages(poison=0.5)
    c = _cache(dev, k0, v0)
    n = hq + 2 * hkv
    cat = (s.randn(s.T, n * dim) * 2).to(DTYPES[src])
    q, k, v = (x.unflatten(1, (-1, dim)) for x in cat.split([hq * dim, hkv * dim, hkv * dim], 1))
    g = cat.to(dev)
    gq, gk, gv = (x.unflatten(1, (-1, dim)) for x in g.split([hq * dim, hkv * dim, hkv * dim], 1))
    qn = 1 + 0.3 * s.randn(dim) if norm else None
    kn = 1 + 0.3 * s.randn(dim) if norm else None
    rope = HipRotary(dim, base=1e6, rotary_dim=rot, interleaved=inter, attn_factor=1.1, device=dev) if rot else None
    inv = 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    out = torch.full((s.T, hq, dim), 5.0, dtype=s.dtype, device=dev)
    got = c.append(gq, gk, gv, s.batch(dev), rope, None if qn is None else qn.to(dev), None if kn is None else kn.to(dev),
                   out=out).cpu()
    N = s.q_start[-1]
    pos, place = torch.zeros(N), []
    for b, (m, ln) in enumerate(zip(s.q_lens, s.lens)):
        for i in range(m):
            j = ln - m + i
            pos[s.q_start[b] + i] = s.prefix + j
            place.append((int(s.table[b, j // 16]), j % 16))
    half = HALF_STEP[s.dtype]

    def check(y, x, w, what):
        ref, mag = rotate_reference(norm_reference(x[:N], w), pos, inv, inter, 1.1 if rot else 1.0)
        # half a step of the result; the norm's sums, root and products and the rotation's angle, cosine
        # and products: under 32 roundings of 2^-24 of the pair's magnitudes; 2^-25: fp16 below its range
        tol = half * ref.abs() + 32 * 2.0 ** -24 * mag + 2.0 ** -25
        d = (y[:N].double() - ref).abs()
        assert bool((d <= tol).all()), (what, float((d - tol).max()))

    check(got, q, qn, "q")
    pg, ro = (torch.tensor(x) for x in zip(*place))
    ck, cv = c.k.cpu(), c.v.cpu()
    check(ck[pg, :, ro], k, kn, "k")
    assert torch.equal(cv[pg, :, ro], v[:N].to(s.dtype))
    ck[pg, :, ro], cv[pg, :, ro] = k0[pg, :, ro], v0[pg, :, ro]
    assert torch.equal(ck, k0) and torch.equal(cv, v0), "rows of other tokens changed"
    assert bool((got[N:] == 5.0).all())


def test_append_far_positions(dev):
    """Positions of millions: the angle is formed and reduced in float64."""
    log("append far positions")
    from pgmoe import HipPagedKVCache, HipRotary, KVBatch
    c = HipPagedKVCache(2, 256, 1, 128, device=dev)
    inv = 1e4 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    g = torch.Generator().manual_seed(3)
    for prefix in (1 << 20, (1 << 23) + 1, 1 << 29):
        pages = torch.zeros(-(-prefix // 256), dtype=torch.int32, device=dev)  # not read by append
        b = KVBatch([[0], [1]], [5, 200], prefix_pages=pages, prefix_len=prefix, device=dev)
        q = torch.randn(2, 2, 128, generator=g)
        got = c.append(q.to(dev), q[:, :1].to(dev), q[:, :1].to(dev), b, HipRotary(128, device=dev)).cpu().double()
        ref, mag = rotate_reference(q, torch.tensor([prefix + 4, prefix + 199]), inv, False)
        assert bool(((got - ref).abs() <= 2.0 ** -11 * ref.abs() + 16 * 2.0 ** -24 * mag + 2.0 ** -25).all()), prefix


def test_append_skips_what_has_no_place(dev):
    """Bad page ids, rows past the table and negative own indexes: the query is made, nothing is written."""
    log("append bad pages")
    from pgmoe import HipPagedKVCache, KVBatch
    c = HipPagedKVCache(4, 16, 2, 64, dtype=torch.bfloat16, device=dev)
    x = torch.randn(9, 2, 64, device=dev)
    for table, lens, qs in (([[-1]], [9], [0, 9]), ([[4]], [9], [0, 9]), ([[2 ** 31 - 1]], [9], [0, 9]),
                            ([[3]], [2 ** 31 - 1], [0, 9]), ([[1]], [0], [0, 9])):
        got = c.append(x, x, x, KVBatch(torch.tensor(table, dtype=torch.int64).to(torch.int32), lens, q_start=qs, device=dev))
        assert torch.equal(got, x.to(torch.bfloat16))
        assert int(torch.count_nonzero(c.k)) == 0 and int(torch.count_nonzero(c.v)) == 0
    c.append(x, x, x, KVBatch([[1]], [4], q_start=[0, 9], device=dev))  # own indexes -5 .. 3
    assert torch.equal(c.k[1, :, :4], x[5:].transpose(0, 1).to(torch.bfloat16))
    assert int(torch.count_nonzero(c.k[1, :, 4:])) == 0 and int(torch.count_nonzero(c.k[0])) == 0


def test_append_refusals(dev):
    from pgmoe import HipPagedKVCache, HipRotary, KVBatch
    c = HipPagedKVCache(4, 16, 2, 64, device=dev)
    b = KVBatch([[0], [1]], [1, 1], device=dev)
    q, k = torch.zeros(2, 4, 64, device=dev), torch.zeros(2, 2, 64, device=dev)
    with pytest.raises(ValueError, match="dtype"):
        c.append(q, k.half(), k, b)
    with pytest.raises(ValueError):
        c.append(q, k[:1], k, b)
    with pytest.raises(ValueError):
        c.append(q, q, q, b)  # 4 KV heads
    with pytest.raises(ValueError, match="head_dim"):
        c.append(q, k, k, b, HipRotary(128, device=dev))
    with pytest.raises(ValueError, match="q_norm"):
        c.append(q, k, k, b, q_norm=torch.ones(32, device=dev))
    with pytest.raises(NotImplementedError):
        c.append(q.double(), k.double(), k.double(), b)
    with pytest.raises(ValueError, match="out"):
        c.append(q, k, k, b, out=torch.zeros(2, 4, 64, device=dev))
