"""float64 references and inputs for the paged KV cache, attention and sampling tests."""

from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import List, Optional

import numpy as np
import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@dataclass
class Step:
    """One call's sequences on the host: q tokens, own keys, page tables; `extra` token rows behind them."""
    q_lens: List[int]
    lens: List[int]
    hq: int
    hkv: int
    dim: int
    page: int = 16
    prefix: int = 0
    extra: int = 0
    dtype: torch.dtype = torch.float16
    seed: int = 0
    spare_pages: int = 2
    table: torch.Tensor = field(init=False)

    def __post_init__(self):
        g = torch.Generator().manual_seed(self.seed)
        self.gen = g
        self.q_start = [sum(self.q_lens[:i]) for i in range(len(self.q_lens) + 1)]
        self.T = self.q_start[-1] + self.extra
        pages = [max(1, -(-n // self.page)) for n in self.lens]
        shared = -(-self.prefix // self.page)
        self.n_pages = sum(pages) + shared + self.spare_pages
        order = torch.randperm(self.n_pages, generator=g, dtype=torch.int32)
        self.prefix_pages = order[:shared].clone()
        self.table = torch.full((len(self.lens), max(pages)), -1, dtype=torch.int32)  # past a sequence: no page
        at = shared
        for b, n in enumerate(pages):
            self.table[b, :n] = order[at:at + n]
            at += n

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.gen)

    def pages(self, poison: float = float("nan")):
        """K and V pages: normal values where a key lies, `poison` in every other row."""
        shape = (self.n_pages, self.hkv, self.page, self.dim)
        k, v = self.randn(*shape).to(self.dtype), self.randn(*shape).to(self.dtype)
        used = torch.zeros(self.n_pages, self.page, dtype=torch.bool)
        for j in range(self.prefix):
            used[int(self.prefix_pages[j // self.page]), j % self.page] = True
        for b, n in enumerate(self.lens):
            for j in range(n):
                used[int(self.table[b, j // self.page]), j % self.page] = True
        dead = ~used[:, None, :, None].expand(shape)
        k[dead], v[dead] = poison, poison
        return k, v

    def q(self, scale: float = 1.0):
        return (self.randn(self.T, self.hq, self.dim) * scale).to(self.dtype)

    def batch(self, dev, ragged: Optional[bool] = None):
        from pgmoe import KVBatch
        ragged = self.extra > 0 or any(n != 1 for n in self.q_lens) if ragged is None else ragged
        return KVBatch(self.table.to(dev), torch.tensor(self.lens, dtype=torch.int32, device=dev),
                       q_start=torch.tensor(self.q_start, dtype=torch.int32, device=dev) if ragged else None,
                       prefix_pages=self.prefix_pages.to(dev) if self.prefix else None, prefix_len=self.prefix)

    def keys(self, b: int, n: int, pages: torch.Tensor, head: int) -> torch.Tensor:
        """The prefix's rows and sequence b's first n own rows, float64 [prefix + n, dim]."""
        at = [(int(self.prefix_pages[j // self.page]), j % self.page) for j in range(self.prefix)]
        at += [(int(self.table[b, j // self.page]), j % self.page) for j in range(n)]
        if not at:
            return torch.zeros(0, self.dim, dtype=torch.float64)
        p, r = (torch.tensor(x) for x in zip(*at))
        return pages[p, head, r].double()


def attend_reference(s: Step, q, k, v, scale: Optional[float] = None):
    """(out, lse, tolerance of out, tolerance of lse) in float64; rows behind the last sequence NaN.

    Tolerance, from the arithmetic the entry point documents: the result rounded once (half a step of
    |out|); every probability rounded once to the cache's type and sums of n terms in fp32, relative to
    the sum of their magnitudes A = sum p |v| / sum p; a score's fp32 sum over D products is off by
    2^-24 (D + 4) sum |q k| scale at most, plus three roundings of the score itself, and moves p by
    as much, in numerator and denominator."""
    scale = s.dim ** -0.5 if scale is None else scale
    out = torch.full((s.T, s.hq, s.dim), math.nan, dtype=torch.float64)
    tol = torch.zeros_like(out)
    lse = torch.full((s.T, s.hq), math.nan, dtype=torch.float64)
    ltol = torch.zeros_like(lse)
    g, half, unit = s.hq // s.hkv, HALF_STEP[s.dtype], 2.0 ** -24
    for b, (n, ln) in enumerate(zip(s.q_lens, s.lens)):
        for h in range(s.hkv):
            kk, vv = s.keys(b, ln, k, h), s.keys(b, ln, v, h)
            qq = q[s.q_start[b]:s.q_start[b + 1], h * g:(h + 1) * g].double()
            for i in range(n):
                see = s.prefix + max(0, ln - n + i + 1)
                t = s.q_start[b] + i
                if see == 0:
                    out[t, h * g:(h + 1) * g] = 0
                    lse[t, h * g:(h + 1) * g] = -math.inf
                    continue
                x = qq[i] @ kk[:see].T * scale
                w = torch.softmax(x, -1)
                o = w @ vv[:see]
                mag = (qq[i].abs() @ kk[:see].abs().T * scale).amax(-1, keepdim=True)
                ds = unit * ((s.dim + 4) * mag + 3 * x.abs().amax(-1, keepdim=True))
                a = w @ vv[:see].abs()
                out[t, h * g:(h + 1) * g] = o
                tol[t, h * g:(h + 1) * g] = half * o.abs() + a * (1.01 * half + 2 * ds + 2 * (see + 64) * unit) + 2.0 ** -25
                ll = torch.logsumexp(x, -1)
                lse[t, h * g:(h + 1) * g] = ll
                ltol[t, h * g:(h + 1) * g] = (ds[:, 0] + (see + 64) * unit) + 4 * unit * ll.abs()
    return out, lse, tol, ltol


def check_attend(s: Step, got, ref, lse=None):
    out, rl, tol, ltol = ref
    n = s.q_start[-1]
    d = (got[:n].double().cpu() - out[:n]).abs()
    bad = ~(d <= tol[:n])
    assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} values off, first at "
                                 f"{bad.nonzero()[0].tolist()}: {d[bad][0]:.3e} > {tol[:n][bad][0]:.3e}")
    if lse is not None:
        g, r = lse[:n].double().cpu(), rl[:n]
        empty = torch.isinf(r)
        assert torch.equal(torch.isinf(g) & (g < 0), empty)
        assert bool(((g - r).abs()[~empty] <= ltol[:n][~empty]).all()), (g - r).abs()[~empty].max()


def rotate_reference(x, pos, inv_freq, interleaved, attn_factor=1.0):
    """float64 rotation of x [T, H, D] at positions pos [T]; the rotated pairs' magnitudes beside it."""
    x = x.double().clone()
    half = inv_freq.numel()
    a = pos.double()[:, None] * inv_freq.double()
    c, s = (a.cos() * attn_factor)[:, None], (a.sin() * attn_factor)[:, None]
    i1 = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    i2 = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    p, q = x[..., i1].clone(), x[..., i2].clone()
    mag = x.abs()
    x[..., i1], x[..., i2] = p * c - q * s, q * c + p * s
    mag[..., i1] = mag[..., i2] = (p.abs() + q.abs()) * abs(attn_factor)
    return x, mag


def norm_reference(x, w, eps=1e-6):
    x = x.double()
    return x if w is None else x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def sample_reference(x, u, temperature, top_k, top_p, min_p):
    """Token and log-probability of one row, float64."""
    x = np.asarray(x, dtype=np.float64)
    ok = x > -np.inf
    if not ok.any():
        return -1, -math.inf
    x = np.where(ok, x, -np.inf)
    if temperature <= 0:
        return int(np.argmax(x)), 0.0
    m = x.max()
    if np.isinf(m):
        e = (x == m).astype(np.float64)
    else:
        e = np.where(ok, np.exp((np.where(ok, x, m) - m) / temperature), 0.0)
    order = np.lexsort((np.arange(len(x)), -x))
    n = len(x)
    if top_k > 0:
        n = min(n, top_k)
    if top_p < 1:
        cum = np.cumsum(e[order])
        n = min(n, int((cum - e[order] < top_p * cum[-1]).sum()))
    if min_p > 0:
        n = min(n, int((e >= min_p).sum()))
    kept = np.zeros(len(x))
    kept[order[:max(1, n)]] = e[order[:max(1, n)]]
    c = np.cumsum(kept)
    at = int((c <= u * c[-1]).sum())
    at = min(at, int(np.nonzero(kept)[0].max()))
    return at, math.log(kept[at] / c[-1])
