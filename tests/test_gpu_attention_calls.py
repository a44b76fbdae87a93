"""What HipPagedKVCache, KVBatch and HipRotary accept, refuse and keep from call to call."""

import pytest

from gpu_helpers import log
from kv_helpers import Step, attend_reference, check_attend

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda", 0)


def _made(dev, **kw):
    from pgmoe import HipPagedKVCache
    s = Step([1, 1], [40, 70], 8, 2, 128, 16, seed=1, **kw)
    k, v = s.pages()
    q = s.q()
    return s, HipPagedKVCache.from_tensors(k.to(dev), v.to(dev)), q.to(dev), attend_reference(s, q, k, v)


def test_page_tables_whose_rows_overlap_are_refused(dev):
    from pgmoe import KVBatch
    log("page table rows that overlap")
    row = torch.zeros(1, 4, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="overlap"):
        KVBatch(row.expand(2, 4), [4, 5])
    with pytest.raises(ValueError, match="overlap"):
        KVBatch(torch.zeros(9, dtype=torch.int32, device=dev).as_strided((2, 4), (3, 1)), [4, 5])
    KVBatch(row.expand(1, 4), [4])  # a single row overlaps nothing


def test_a_refused_call_leaves_the_next_ones(dev):
    """A batch that the library refuses, then a valid one of the same shape on the same cache."""
    log("attend after a refusal")
    s, c, q, ref = _made(dev)
    b = s.batch(dev)
    stride, b._c.table_stride = b._c.table_stride, 0
    with pytest.raises(RuntimeError, match="overlap"):
        c.attend(q, b)
    b._c.table_stride = stride
    check_attend(s, c.attend(q, b), ref)


def test_nothing_is_kept_for_a_call_s_sizes(dev):
    """Calls of ever new sizes leave the cache object as it was."""
    from pgmoe import KVBatch
    log("attend of many sizes")
    s, c, q, _ = _made(dev)

    def held():
        return {n: len(x) for n, x in vars(c).items() if hasattr(x, "__len__") and not isinstance(x, torch.Tensor)}

    before = held()
    for T in range(1, 20):
        c.attend(torch.zeros(T, 8, 128, dtype=s.dtype, device=dev),
                 KVBatch(s.table.to(dev), s.lens, q_start=[0, T, T], prefix_pages=[0, 1], prefix_len=T))
    assert held() == before


def test_what_a_call_holds_as_it_was_given_is_read_only(dev):
    """The kernels read the numbers a batch, a cache and a rotary were made with: another value is refused, and the
    next call computes what it did before."""
    from pgmoe import HipRotary
    log("read-only numbers")
    s, c, q, ref = _made(dev, prefix=20)
    b, rope = s.batch(dev), HipRotary(128, rotary_dim=64, device=dev)
    for x, names in ((b, ("n_seqs", "max_pages", "prefix_len", "device")),
                     (c, ("n_pages", "n_kv_heads", "page_size", "head_dim", "dtype", "device")),
                     (rope, ("head_dim", "rotary_dim", "interleaved", "attn_factor", "turns", "device"))):
        for n in names:
            was = getattr(x, n)
            with pytest.raises(AttributeError):
                setattr(x, n, was)
            assert getattr(x, n) is was or getattr(x, n) == was
    assert (b.n_seqs, b.max_pages, b.prefix_len) == (2, 5, 20)
    assert (c.n_pages, c.n_kv_heads, c.page_size, c.head_dim, c.dtype) == (s.n_pages, 2, 16, 128, s.dtype)
    assert (rope.head_dim, rope.rotary_dim, rope.interleaved, rope.attn_factor) == (128, 64, False, 1.0)
    check_attend(s, c.attend(q, b), ref)


@pytest.mark.parametrize("seqs,tokens,prefix", [(3, 40, 0), (300, 64, 20), (2048, 4096, 0)])
def test_a_q_start_that_decreases_stays_inside(dev, seqs, tokens, prefix):
    """Sequences that all claim every token, on the device where the host does not see it (together they are more work than
    32 bits count): nothing behind the call's rows changes, and the next call is as ever."""
    from pgmoe import HipPagedKVCache, KVBatch
    log(f"attend q_start up and down, {seqs} sequences of {tokens} tokens, prefix {prefix}")
    c = HipPagedKVCache(40, 256, 8, 64, device=dev)
    up_down = torch.tensor([tokens * (i % 2) for i in range(seqs + 1)], dtype=torch.int32, device=dev)
    table = torch.zeros(seqs, 256, dtype=torch.int32, device=dev)
    b = KVBatch(table, torch.full((seqs,), 65536, dtype=torch.int32, device=dev), q_start=up_down,
                prefix_pages=torch.zeros(1, dtype=torch.int32, device=dev), prefix_len=prefix)
    buf = torch.full((tokens + 8, 64, 64), 3.0, dtype=torch.float16, device=dev)
    k = c.k.clone()
    c.attend(torch.zeros(tokens, 64, 64, dtype=torch.float16, device=dev), b, out=buf[:tokens])
    torch.cuda.synchronize()
    assert bool((buf[tokens:] == 3.0).all()) and torch.equal(c.k, k)
    s, c, q, ref = _made(dev, prefix=20)
    check_attend(s, c.attend(q, s.batch(dev)), ref)


def test_strides_of_axes_of_one_element_mean_nothing(dev):
    """One page, one KV head, one sequence: views whose strides there are odd are as good as any."""
    from pgmoe import HipPagedKVCache, KVBatch
    log("strides of single elements")
    g = torch.Generator(dev).manual_seed(1)
    k, v = (torch.randn(1, 1, 16, 64, generator=g, device=dev).half() for _ in range(2))
    q = torch.randn(1, 2, 64, generator=g, device=dev).half()
    want = HipPagedKVCache.from_tensors(k, v).attend(q, KVBatch([[0]], [9], device=dev))
    odd = k.as_strided(k.shape, (3, 5, 64, 1))
    other = v.as_strided(v.shape, (1, 1, 64, 1))
    c = HipPagedKVCache.from_tensors(odd, other)
    table = torch.zeros(7, 3, dtype=torch.int32, device=dev)
    lens = torch.full((7,), 9, dtype=torch.int32, device=dev)
    assert torch.equal(c.attend(q, KVBatch(table[:1, :1], lens.as_strided((1,), (4,)))), want)
    assert torch.equal(c.attend(q, KVBatch(table.t()[:1, :1], lens[:1])), want)
    with pytest.raises(ValueError):
        KVBatch(table.t()[:2], lens[:2])


def test_sizes_past_32_bits_are_refused(dev):
    """Before they become another number on the way into the library."""
    from pgmoe import KVBatch, sample_tokens
    log("sizes past 32 bits")
    one = torch.zeros(1, dtype=torch.int32, device=dev)
    for n in (2 ** 30 + 1, 2 ** 32, 2 ** 32 + 5):
        with pytest.raises(NotImplementedError, match="prefix_len"):
            KVBatch([[0]], [1], prefix_pages=one, prefix_len=n, device=dev)
    with pytest.raises(NotImplementedError, match="rows"):
        sample_tokens(torch.zeros(1, 1, device=dev).expand(2 ** 32 + 2, 1), torch.zeros(1, device=dev).expand(2 ** 32 + 2))
    with pytest.raises(NotImplementedError, match="rows"):
        sample_tokens(torch.zeros(1, 1, device=dev).expand(2 ** 22 + 1, 1), torch.zeros(1, device=dev).expand(2 ** 22 + 1))
