"""Paged KV cache with rotary append and shared-prefix attention (pgmoe_rope_append, pgmoe_attend).

The step between a layer's Q/K/V projections (FusedLinearPack) and its output projection:

    rope  = HipRotary(head_dim, base=1e6)
    cache = HipPagedKVCache(n_pages, page_size, n_kv_heads, head_dim)      # one a layer
    batch = KVBatch(page_table, lens, q_start=..., prefix_pages=..., prefix_len=...)   # one a step, all layers
    q = cache.append(q, k, v, batch, rope, q_norm=..., k_norm=...)   # norms + rotary + K/V rows, rotated q
    o = cache.attend(q, batch)                                       # softmax(q K^T / sqrt(D)) V

Every sequence sees the ``prefix_len`` keys of ``prefix_pages`` (a system prompt, a document) and then
its own keys; the prefix's keys and values are read for 128 query rows of a KV head at a time, whichever
sequences they belong to.  The batch's tensors live on the device and are read when the kernels run: a
program updates them in place between steps (``lens.add_(1)`` on the calls' stream, or ordered with it),
and a captured graph replays on what they then hold (keep cache, batch, rotary and norm weights as long
as the graph).  Nothing synchronises with the host but the constructors.  There is no CPU path: CPU
tensors, and types, widths and page sizes without a kernel, raise.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Tuple, Union

import torch

from ._lib import KVBatch as _KVBatch
from ._lib import KVCache as _KVCache
from ._lib import check, lib

_DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_CACHE_DT = (torch.float16, torch.bfloat16)
_DIMS = (64, 128, 256)
_PAGES = (16, 32, 64, 128, 256)
_MAX_SEQS = 4096
_MAX_KEYS = 1 << 30  # of a prefix, and of one sequence

_IntTensor = Union[torch.Tensor, Sequence[int]]


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def launch(dev: torch.device, what: str, fn, *args) -> None:
    """fn(*args, stream) of the C ABI on `dev`'s current stream, with `dev` the current device; raises on a
    status other than 0.  (The stream's handle by itself: a Stream object costs 2 us more.)"""
    stream = _raw_stream(dev.index) if _raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream
    if torch.cuda.current_device() == dev.index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream)
    if rc:
        check(rc, what)


def _cuda_device(device: Optional[Union[torch.device, str]]) -> torch.device:
    dev = torch.device("cuda" if device is None else device)
    if dev.type != "cuda":
        raise ValueError("pgmoe attention runs on a HIP device (torch.device('cuda', i))")
    return torch.device("cuda", torch.cuda.current_device()) if dev.index is None else dev


class HipRotary:
    """Rotary positions: pair i turns by position * inv_freq[i] radians.

    inv_freq: float64 [rotary_dim / 2], or None for base ** (-2 i / rotary_dim).  freq_factors (a
    GGUF file's rope_freqs) divide it, position_scale multiplies every position (linear scaling),
    attn_factor scales cosine and sine (YaRN).  Pairs are (i, i + rotary_dim / 2), or (2 i, 2 i + 1)
    with interleaved."""

    def __init__(self, head_dim: int, base: float = 10000.0, rotary_dim: Optional[int] = None,
                 interleaved: bool = False, inv_freq: Optional[torch.Tensor] = None,
                 freq_factors: Optional[torch.Tensor] = None, position_scale: float = 1.0, attn_factor: float = 1.0,
                 device: Optional[Union[torch.device, str]] = None) -> None:
        if inv_freq is not None:
            if inv_freq.dim() != 1 or (rotary_dim is not None and inv_freq.numel() * 2 != rotary_dim):
                raise ValueError("inv_freq holds one float64 frequency a pair (rotary_dim / 2)")
            rotary_dim = 2 * inv_freq.numel()
            if device is None:
                device = inv_freq.device if inv_freq.device.type == "cuda" else None
        rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
        if rotary_dim < 16 or rotary_dim > head_dim or rotary_dim % 16:
            raise ValueError(f"rotary_dim {rotary_dim}: a multiple of 16 up to head_dim {head_dim}")
        if not (math.isfinite(position_scale) and math.isfinite(attn_factor) and base > 0):
            raise ValueError("base must be positive, position_scale and attn_factor finite")
        self._device = _cuda_device(device)
        self._head_dim, self._rotary_dim, self._interleaved = int(head_dim), rotary_dim, bool(interleaved)
        self._attn_factor = float(attn_factor)
        if inv_freq is None:
            inv_freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
        f = inv_freq.to("cpu", torch.float64)
        if freq_factors is not None:
            if freq_factors.numel() != rotary_dim // 2:
                raise ValueError("freq_factors holds one factor a pair (rotary_dim / 2)")
            f = f / freq_factors.to("cpu", torch.float64).reshape(-1)
        self._turns = (f * (position_scale / (2.0 * math.pi))).to(self._device)

    # as they were given: the kernel reads rotary_dim / 2 turns
    device = property(lambda self: self._device)
    head_dim = property(lambda self: self._head_dim)
    rotary_dim = property(lambda self: self._rotary_dim)
    interleaved = property(lambda self: self._interleaved)
    attn_factor = property(lambda self: self._attn_factor)
    turns = property(lambda self: self._turns)


class KVBatch:
    """The sequences of one step (pgmoe_kv_batch): `page_table` int32 [n_seqs, max_pages], `lens`
    int32 [n_seqs] (own keys of each sequence, this step's among them), `q_start` int32 [n_seqs + 1]
    (first token row of each sequence and the end; None: one token each), `prefix_pages` int32 and
    `prefix_len` (keys every sequence sees before its own).

    Tensors on the device are kept, not copied, and may be updated in place.  Lists and CPU tensors
    are checked and copied to the device.  The numbers (n_seqs, max_pages, prefix_len) are the batch's for
    good: a step behind another prefix takes another batch."""

    def __init__(self, page_table: _IntTensor, lens: _IntTensor, q_start: Optional[_IntTensor] = None,
                 prefix_pages: Optional[_IntTensor] = None, prefix_len: int = 0,
                 device: Optional[Union[torch.device, str]] = None) -> None:
        given = [t for t in (page_table, lens, q_start, prefix_pages)
                 if isinstance(t, torch.Tensor) and t.device.type == "cuda"]
        self._device = given[0].device if given else _cuda_device(device)
        self._table = self._int32("page_table", page_table, 2, -1)
        self._lens = self._int32("lens", lens, 1, 0)
        n = self._table.shape[0]
        if not 1 <= n <= _MAX_SEQS:
            raise NotImplementedError(f"{n} sequences (1 .. {_MAX_SEQS})")
        if self._table.shape[1] < 1 or self._lens.shape[0] != n:
            raise ValueError(f"page_table {tuple(self._table.shape)} and lens {tuple(self._lens.shape)} of {n} sequences")
        if n > 1 and self._table.stride(0) < self._table.shape[1]:
            raise ValueError("the rows of page_table overlap")
        self._q_start = None
        if q_start is not None:
            self._q_start = self._int32("q_start", q_start, 1, 0)
            if self._q_start.shape[0] != n + 1:
                raise ValueError(f"q_start holds {self._q_start.shape[0]} rows, {n} sequences need {n + 1}")
            host = q_start if not isinstance(q_start, torch.Tensor) else q_start.tolist() if q_start.device.type == "cpu" else None
            if host is not None and (host[0] != 0 or any(a > b for a, b in zip(host, host[1:]))):
                raise ValueError("q_start begins at 0 and does not decrease")
        self._prefix_len = int(prefix_len)
        if self._prefix_len < 0:
            raise ValueError("negative prefix_len")
        if self._prefix_len > _MAX_KEYS or self._table.shape[1] > _MAX_KEYS // _PAGES[0]:
            raise NotImplementedError(f"prefix_len {prefix_len}, {self._table.shape[1]} pages a sequence (up to {_MAX_KEYS} keys)")
        self._prefix = None if prefix_pages is None else self._int32("prefix_pages", prefix_pages, 1, -1)
        if self._prefix_len and self._prefix is None:
            raise ValueError("prefix_len without prefix_pages")
        self._n_seqs, self._max_pages = n, int(self._table.shape[1])
        self._c = _KVBatch(self._table.data_ptr(), self._lens.data_ptr(),
                           None if self._q_start is None else self._q_start.data_ptr(),
                           None if self._prefix is None else self._prefix.data_ptr(),
                           self._table.stride(0), n, self._max_pages, self._prefix_len)
        self._ref = ctypes.byref(self._c)

    def _int32(self, name: str, x: _IntTensor, dims: int, least: int) -> torch.Tensor:
        t = x if isinstance(x, torch.Tensor) else torch.tensor(x, dtype=torch.int32)
        if t.dim() != dims:
            raise ValueError(f"{name} has {t.dim()} dimensions, not {dims}")
        if t.device.type != "cuda":
            if t.is_floating_point() or (t.numel() and (int(t.min()) < least or int(t.max()) > 2 ** 31 - 1)):
                raise ValueError(f"{name} holds int32 values from {least} on")
            return t.to(self._device, torch.int32).contiguous()
        if t.dtype != torch.int32:
            raise ValueError(f"{name} is an int32 tensor")
        if t.device != self._device:
            raise ValueError(f"{name} is on {t.device}, the batch on {self._device}")
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name} must be contiguous along its rows")
        return t

    # the tensors the kernels read: updated in place, never replaced (the addresses are fixed)
    page_table = property(lambda self: self._table)
    lens = property(lambda self: self._lens)
    q_start = property(lambda self: self._q_start)
    prefix_pages = property(lambda self: self._prefix)
    device = property(lambda self: self._device)
    # numbers that calls and captured graphs hold as they were given: another value is another batch
    n_seqs = property(lambda self: self._n_seqs)
    max_pages = property(lambda self: self._max_pages)
    prefix_len = property(lambda self: self._prefix_len)


class HipPagedKVCache:
    """K and V pages of one attention layer: [n_pages, n_kv_heads, page_size, head_dim] each."""

    def __init__(self, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.float16, device: Optional[Union[torch.device, str]] = None) -> None:
        dev = _cuda_device(device)
        self._check(n_pages, page_size, n_kv_heads, head_dim, dtype)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a KV cache is made before a graph is captured: each replay would clear its pages")
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        self._bind(torch.zeros(shape, dtype=dtype, device=dev), torch.zeros(shape, dtype=dtype, device=dev))
        torch.cuda.current_stream(dev).synchronize()  # cleared before any other stream writes to them

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor) -> "HipPagedKVCache":
        """A cache over existing pages, views of a larger allocation among them (a layer's slice, K and
        V interleaved): both [n_pages, n_kv_heads, page_size, head_dim] with the same strides, the last
        dimension contiguous, the others in multiples of 8 elements."""
        self = cls.__new__(cls)
        same = k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and k.device == v.device
        if not same or cls._strides(k) != cls._strides(v):
            raise ValueError("k and v pages: [n_pages, n_kv_heads, page_size, head_dim] of one type, device and layout")
        if k.device.type != "cuda":
            raise ValueError("pgmoe attention runs on a HIP device tensor")
        n, h, ps, d = k.shape
        self._check(n, ps, h, d, k.dtype)
        st = cls._strides(k)
        if st[3] != 1 or any(x % 8 for x in st[:3]) or k.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError("pages need a contiguous head_dim, strides of whole 16 bytes and 16-byte alignment")
        if st[2] < d or st[2] > 1 << 22 or any(s <= 0 for s, m in zip(st, k.shape) if m > 1):
            raise ValueError("the rows of a page overlap or lie too far apart")
        self._bind(k, v)
        return self

    @staticmethod
    def _strides(x: torch.Tensor) -> Tuple[int, ...]:
        """x's strides; 0 of an axis of one element, whose stride means nothing."""
        return tuple(s if m > 1 else 0 for s, m in zip(x.stride(), x.shape))

    @staticmethod
    def _check(n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, dtype: torch.dtype) -> None:
        if dtype not in _CACHE_DT:
            raise NotImplementedError(f"KV cache of dtype {dtype} (fp16 or bf16)")
        if head_dim not in _DIMS:
            raise NotImplementedError(f"head_dim {head_dim} (one of {_DIMS})")
        if page_size not in _PAGES:
            raise NotImplementedError(f"page_size {page_size} (one of {_PAGES})")
        if not (1 <= n_pages < 2 ** 31 and 1 <= n_kv_heads <= 1024):
            raise ValueError(f"{n_pages} pages of {n_kv_heads} KV heads")

    def _bind(self, k: torch.Tensor, v: torch.Tensor) -> None:
        lib()
        self._k, self._v = k, v
        self._n_pages, self._n_kv_heads, self._page_size, self._head_dim = (int(x) for x in k.shape)
        self._dtype, self._device = k.dtype, k.device
        st = self._strides(k)
        self._c = _KVCache(k.data_ptr(), v.data_ptr(), st[0], st[1], st[2], self._n_pages, self._page_size,
                           self._n_kv_heads, self._head_dim, _DT[k.dtype])
        self._ref = ctypes.byref(self._c)

    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    n_pages = property(lambda self: self._n_pages)
    n_kv_heads = property(lambda self: self._n_kv_heads)
    page_size = property(lambda self: self._page_size)
    head_dim = property(lambda self: self._head_dim)
    dtype = property(lambda self: self._dtype)
    device = property(lambda self: self._device)

    # ------------------------------------------------------------------ checks
    def _heads(self, name: str, x: torch.Tensor, dtypes, heads: Optional[int] = None) -> Tuple[torch.Tensor, int, int]:
        """x checked, and its token and head strides; copied where its rows cannot be read 16 bytes at a time."""
        shape, dtype = x.shape, x.dtype
        if x.device != self._device:
            raise ValueError(f"{name} is on {x.device}, the cache on {self._device}")
        if dtype not in dtypes:
            raise NotImplementedError(f"{name} of dtype {dtype}")
        if len(shape) != 3 or shape[2] != self._head_dim or (heads is not None and shape[1] != heads):
            raise ValueError(f"{name} {tuple(shape)}: [tokens, {'heads' if heads is None else heads}, {self._head_dim}]")
        a, b, c = x.stride()
        if c != 1 or (a | b) & (3 if dtype is torch.float32 else 7) or x.data_ptr() & 15:
            x = x.clone(memory_format=torch.contiguous_format)
            a, b, c = x.stride()
        return x, a, b

    def _tokens(self, q: torch.Tensor, batch: KVBatch) -> Tuple[int, int]:
        T, hq, _ = q.shape
        if hq < 1 or hq % self._n_kv_heads:
            raise ValueError(f"{hq} query heads on {self._n_kv_heads} KV heads")
        if batch._device != self._device:
            raise ValueError(f"the batch is on {batch.device}, the cache on {self._device}")
        if batch._q_start is None and T != batch._n_seqs:
            raise ValueError(f"{T} tokens of {batch.n_seqs} sequences: q_start says which are whose")
        if batch._prefix_len > (0 if batch._prefix is None else batch._prefix.shape[0]) * self._page_size:
            raise ValueError(f"a prefix of {batch.prefix_len} keys on {batch._prefix.shape[0]} pages of {self._page_size}")
        return T, hq

    def _out(self, out: Optional[torch.Tensor], T: int, hq: int) -> torch.Tensor:
        if out is None:
            return torch.empty((T, hq, self._head_dim), dtype=self._dtype, device=self._device)
        if out.shape != (T, hq, self._head_dim) or out.dtype != self._dtype or out.device != self._device:
            raise ValueError(f"out: [{T}, {hq}, {self._head_dim}] of {self._dtype} on {self._device}")
        if not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("out must be contiguous and 16-byte aligned")
        return out

    @staticmethod
    def _span(t: torch.Tensor) -> Tuple[int, int]:
        n = sum((m - 1) * s for m, s in zip(t.shape, t.stride())) + 1 if t.numel() else 0
        return t.data_ptr(), t.data_ptr() + n * t.element_size()

    def _apart(self, out: torch.Tensor, *others: torch.Tensor) -> None:
        lo, hi = self._span(out)
        for o in others:
            a, b = self._span(o)
            if lo < b and a < hi:
                raise ValueError("out overlaps an input")

    # ------------------------------------------------------------------ operators
    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, batch: KVBatch,
               rope: Optional[HipRotary] = None, q_norm: Optional[torch.Tensor] = None,
               k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Write this step's keys and values into the pages and return the queries, q and k normalised
        (per head, with norm weights [head_dim]) and rotated, in the cache's type [T, n_q_heads, head_dim].

        q [T, n_q_heads, D], k and v [T, n_kv_heads, D]: fp32, fp16 or bf16, all of one type (the parts of
        a fused projection's output as they are).  A token whose page does not exist (an id outside the
        cache, a row past the page table) is not written.  Rows of `out` behind the last sequence are left
        alone.  No two tokens may fall on one cache row."""
        if k.dtype != q.dtype or v.dtype != q.dtype:
            raise ValueError(f"q, k and v of one dtype, not {q.dtype}, {k.dtype}, {v.dtype}")
        q, qt, qh = self._heads("q", q, _DT)
        T, hq = self._tokens(q, batch)
        k, kt, kh = self._heads("k", k, _DT, self._n_kv_heads)
        v, vt, vh = self._heads("v", v, _DT, self._n_kv_heads)
        if k.shape[0] != T or v.shape[0] != T:
            raise ValueError(f"{T} queries, {k.shape[0]} keys, {v.shape[0]} values")
        turns, rot, inter, factor = None, 0, 0, 1.0
        if rope is not None:
            if rope._head_dim != self._head_dim or rope._device != self._device:
                raise ValueError(f"rotary of head_dim {rope.head_dim} on {rope.device}, cache of {self._head_dim} on {self._device}")
            turns, rot, inter, factor = rope._turns.data_ptr(), rope._rotary_dim, rope._interleaved, rope._attn_factor
        qn = None if q_norm is None else self._norm("q_norm", q_norm)
        kn = None if k_norm is None else self._norm("k_norm", k_norm)
        res = self._out(out, T, hq)
        if out is not None:
            self._apart(out, q, k, v, self._k, self._v)
        launch(self._device, "pgmoe_rope_append", lib().pgmoe_rope_append, self._ref, batch._ref, q.data_ptr(), qt, qh,
               k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, _DT[q.dtype], T, hq, turns, rot, inter, factor,
               None if qn is None else qn.data_ptr(), None if kn is None else kn.data_ptr(), eps, res.data_ptr())
        return res

    def _norm(self, name: str, w: torch.Tensor) -> torch.Tensor:
        if w.numel() != self._head_dim or w.device != self._device:
            raise ValueError(f"{name}: {self._head_dim} weights on {self._device}")
        if w.dtype is not torch.float32 or not w.is_contiguous():
            w = w.to(torch.float32).contiguous()
        return w.clone() if w.data_ptr() & 15 else w

    def attend(self, q: torch.Tensor, batch: KVBatch, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
               return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
        """softmax(scale * q K^T) V over the shared prefix and each sequence's own keys up to the query's
        own, in the cache's type [T, n_q_heads, head_dim]; scale defaults to 1 / sqrt(head_dim).  With
        return_lse also log(sum(exp(scale * q K^T))), fp32 [T, n_q_heads].

        q [T, n_q_heads, D] in the cache's type; query head h reads KV head h // (n_q_heads / n_kv_heads).
        A query that sees no key gets zeros and -inf; one that sees a key on a page that does not exist
        gets NaN.  Masked keys and unused page rows may hold anything.  Rows of `out` behind the last
        sequence are left alone.

        Scratch is allocated at every call, for thousands of tokens some hundred MiB to GiB (pgmoe.h).  Single
        tokens behind very long sequences of their own are faster in a call apart from such prompts."""
        q, qt, qh = self._heads("q", q, (self._dtype,))
        T, hq = self._tokens(q, batch)
        scale = self._head_dim ** -0.5 if scale is None else float(scale)
        if not (0.0 < scale < 3e38):
            raise ValueError("scale must be positive and finite")
        res = self._out(out, T, hq)
        if out is not None:
            self._apart(out, q, self._k, self._v)
        lse = torch.empty((T, hq), dtype=torch.float32, device=self._device) if return_lse else None
        # 0 for what pgmoe_attend refuses, which then says why
        n = int(lib().pgmoe_attend_workspace_bytes(self._ref, batch._ref, T, hq))
        # scratch of this call alone, from the stream's allocator: calls on other streams, and graphs that
        # replay side by side, each have their own
        ws = torch.empty(n, dtype=torch.uint8, device=self._device)
        launch(self._device, "pgmoe_attend", lib().pgmoe_attend, self._ref, batch._ref, q.data_ptr(), qt, qh, T, hq, scale,
               res.data_ptr(), None if lse is None else lse.data_ptr(), ws.data_ptr(), n)
        return res if lse is None else (res, lse)
