"""Refusals of the KV cache, attention and sampling entry points, before any device work: the C ABI's
status codes with made-up device addresses, and the Python classes' errors on CPU tensors."""

import ctypes

import pytest
import torch

from pgmoe import _lib


def _cache(**kw):
    c = _lib.KVCache(0x10000, 0x20000, 4 * 16 * 128, 16 * 128, 128, 10, 16, 4, 128, 1)
    for n, v in kw.items():
        setattr(c, n, v)
    return c


def _batch(**kw):
    b = _lib.KVBatch(0x30000, 0x40000, None, None, 8, 3, 8, 0)
    for n, v in kw.items():
        setattr(b, n, v)
    return b


BAD = [
    (dict(dtype=0), {}, -2, "dtype"), (dict(head_dim=96), {}, -2, "head_dim"), (dict(page_size=24), {}, -2, "page_size"),
    (dict(page_size=8), {}, -2, "page_size"), (dict(n_pages=0), {}, -1, "pages"), (dict(k=0x10008), {}, -1, "aligned"),
    (dict(v=None), {}, -1, "aligned"), (dict(row_stride=120), {}, -1, "strides"), (dict(page_stride=8196), {}, -1, "strides"),
    ({}, dict(n_seqs=0), -2, "sequences"), ({}, dict(n_seqs=4097), -2, "sequences"), ({}, dict(lens=None), -1, "NULL"),
    ({}, dict(prefix_len=5), -1, "prefix"), ({}, dict(prefix_len=-1), -1, "prefix"), ({}, dict(max_pages=0), -1, "page table"),
    ({}, dict(table_stride=7), -1, "overlap"), ({}, dict(max_pages=1 << 28, table_stride=1 << 28), -1, "page table"),
]


@pytest.mark.parametrize("cache,batch,code,msg", BAD)
def test_cache_and_batch_are_checked(cache, batch, code, msg):
    L = _lib.lib()
    C, B = _cache(**cache), _batch(**batch)
    assert L.pgmoe_attend(C, B, 0x1000, 4096, 128, 3, 32, 0.1, 0x2000, None, 0x100, 1 << 40, None) == code
    assert msg in L.pgmoe_last_error().decode()
    assert L.pgmoe_attend_workspace_bytes(C, B, 3, 32) == 0
    assert _append(L, C, B) == code
    assert msg in L.pgmoe_last_error().decode()


def _append(L, C, B, q=0x1000, qs=4096, dt=1, T=3, hq=32, turns=0x5000, rot=128, eps=1e-6, out=0x9000, qn=None):
    return L.pgmoe_rope_append(C, B, q, qs, 128, 0x6000, 512, 128, 0x7000, 512, 128, dt, T, hq, turns, rot, 0, 1.0, qn,
                               None, eps, out, None)


def test_append_refusals():
    L = _lib.lib()
    C, B = _cache(), _batch()
    assert _append(L, C, B, T=0) == 0  # nothing to do
    assert _append(L, C, B, dt=7) == -2
    assert _append(L, C, B, rot=24) == -1 and _append(L, C, B, rot=144) == -1 and _append(L, C, B, rot=-16) == -1
    assert _append(L, C, B, q=0x1008) == -1 and _append(L, C, B, qs=4100) == -1 and _append(L, C, B, q=None) == -1
    assert _append(L, C, B, turns=None) == -1 and _append(L, C, B, out=0x9004) == -1 and _append(L, C, B, eps=-1.0) == -1
    assert _append(L, C, B, qn=0x5004) == -1
    assert _append(L, C, B, hq=30) == -1 and _append(L, C, B, T=4) == -1  # 4 tokens of 3 sequences, no q_start
    assert _append(L, None, B) == -1 and _append(L, C, None) == -1


def test_attend_refusals():
    L = _lib.lib()
    C, B = _cache(), _batch()

    def go(q=0x1000, qs=4096, T=3, hq=32, scale=0.1, out=0x2000, ws=0x100, n=1 << 40):
        return L.pgmoe_attend(C, B, q, qs, 128, T, hq, scale, out, None, ws, n, None)

    assert go(T=0) == 0
    assert go(scale=0.0) == -1 and go(scale=float("nan")) == -1 and go(scale=float("inf")) == -1
    assert go(q=None) == -1 and go(q=0x1002) == -1 and go(qs=4100) == -1 and go(out=None) == -1 and go(out=0x2008) == -1
    assert go(T=-1) == -1 and go(hq=0) == -1 and go(hq=34) == -1 and go(T=4) == -1
    assert go(ws=0x110) == -1
    B.q_start = 0x50000
    assert go(T=1 << 24, hq=4 * 64) == -2 and "tokens" in L.pgmoe_last_error().decode()
    B.n_seqs, B.max_pages, B.table_stride = 4096, 1 << 18, 1 << 18  # 4 million keys each of 4096 sequences
    assert go(T=4096) == -2 and "page tables" in L.pgmoe_last_error().decode()
    assert L.pgmoe_attend_workspace_bytes(C, B, 4096, 32) == 0


def test_sample_refusals():
    L = _lib.lib()

    def go(x=0x1000, dt=0, stride=100, rows=2, vocab=100, u=0x2000, S=None, tok=0x3000, **kw):
        S = _lib.Sampling(None, None, None, None, 1.0, 1.0, 0.0, 0) if S is None else S
        for n, v in kw.items():
            setattr(S, n, v)
        return L.pgmoe_sample(x, dt, stride, rows, vocab, u, S, tok, None, 0x100, 1 << 40, None)

    assert go(rows=0) == 0
    assert go(rows=-1) == -1 and go(vocab=0) == -2 and go(vocab=(1 << 20) + 1) == -2 and go(dt=8) == -2
    assert go(x=None) == -1 and go(u=None) == -1 and go(tok=None) == -1 and go(tok=0x3004) == -1 and go(x=0x1002) == -1
    assert go(stride=99) == -1
    for bad in (-1.0, float("nan")):
        assert go(temperature=bad) == -1 and go(top_p=bad) == -1 and go(min_p=bad) == -1
    assert L.pgmoe_sample(0x1000, 0, 100, 2, 100, 0x2000, None, 0x3000, None, None, 0, None) == -1


def test_classes_refuse_cpu_tensors_and_unknown_forms():
    from pgmoe import HipPagedKVCache, HipRotary, KVBatch, sample_tokens
    with pytest.raises(ValueError, match="HIP device"):
        HipPagedKVCache(4, 16, 2, 128, device="cpu")
    with pytest.raises(ValueError, match="HIP device"):
        HipPagedKVCache.from_tensors(torch.zeros(4, 2, 16, 128), torch.zeros(4, 2, 16, 128))
    with pytest.raises(ValueError, match="HIP device"):
        HipRotary(128, device="cpu")
    with pytest.raises(ValueError, match="rotary_dim"):
        HipRotary(128, rotary_dim=40, device="cpu")
    with pytest.raises(ValueError, match="rotary_dim"):
        HipRotary(64, rotary_dim=80, device="cpu")
    with pytest.raises(ValueError, match="HIP device"):
        KVBatch(torch.zeros(2, 3, dtype=torch.int32), [1, 2], device="cpu")
    with pytest.raises(ValueError, match="HIP device"):
        sample_tokens(torch.zeros(2, 10), torch.zeros(2))
    for args, kind in ((((4, 24, 2, 128), {}), "page_size"), (((4, 16, 2, 80), {}), "head_dim"),
                       (((4, 16, 2, 128), dict(dtype=torch.float32)), "dtype")):
        with pytest.raises(NotImplementedError, match=kind):
            HipPagedKVCache._check(*args[0], args[1].get("dtype", torch.float16))


def test_struct_sizes_follow_the_header():
    """The ctypes mirrors' sizes under the C rules of include/pgmoe.h."""
    assert ctypes.sizeof(_lib.KVCache) == 2 * 8 + 3 * 8 + 5 * 4 + 4
    assert ctypes.sizeof(_lib.KVBatch) == 4 * 8 + 8 + 3 * 4 + 4
    assert ctypes.sizeof(_lib.Sampling) == 4 * 8 + 3 * 8 + 4 + 4


def test_sizes_that_no_launch_holds():
    L = _lib.lib()
    C, B = _cache(), _batch(q_start=0x50000)
    assert _append(L, C, B, T=1 << 24) == -2 and "tokens" in L.pgmoe_last_error().decode()
    S = _lib.Sampling(None, None, None, None, 1.0, 1.0, 0.0, 0)
    assert L.pgmoe_sample(0x1000, 0, 2, (1 << 22) + 1, 2, 0x2000, S, 0x3000, None, 0x100, 1 << 60, None) == -2
    assert "rows" in L.pgmoe_last_error().decode()


def test_attend_workspace_without_a_prefix_is_half():
    L = _lib.lib()
    C, B = _cache(), _batch(q_start=0x50000)
    plain = L.pgmoe_attend_workspace_bytes(C, B, 3, 32)
    B.prefix_pages, B.prefix_len = 0x60000, 100
    both = L.pgmoe_attend_workspace_bytes(C, B, 3, 32)
    rows = 3 * 32 * 2 * 4  # both count the slots of both parts
    assert 2 * (plain - rows - 256) <= both - rows <= 2 * (plain - rows + 256)


def test_no_cache_is_made_while_a_graph_is_captured(monkeypatch):
    import torch
    from pgmoe import HipPagedKVCache
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        HipPagedKVCache(4, 16, 1, 64, device="cuda:0")
