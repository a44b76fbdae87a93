"""Decoder-step operators: rotary + paged KV append, attention over a paged cache with a shared
prefix, and token sampling.

Each case is one call of a public entry point of this package (``own`` true) or the same
mathematics in elementary torch operations (``own`` false).  `listed()` holds fixed cases,
`draw(rng)` more of the same ranges, `exact` the float64 result from the definitions.

Head layouts: 32 query heads on 4 or 8 KV heads of 128 and 8 : 1 to 1 : 1 layouts of 64 and 256.
Vocabularies: 151936 (the output head of the package's benchmarks) and smaller ones.
"""

from __future__ import annotations

import math
import os
import random
import sys
from typing import Any, Dict, List

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _pkg() -> Any:
    path = os.path.join(os.getcwd(), "pytorch-engine_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import pgmoe

    return pgmoe


# ------------------------------------------------------------------ cases
def _append(name: str, **kw: Any) -> Dict[str, Any]:
    c = dict(kind="append", batch=1, q_lo=1, q_hi=1, len_lo=1, len_hi=1, prefix=0, page=16, hq=32, hkv=4, dim=128,
             rot=128, interleaved=False, norm=False, src="f16", dtype="f16")
    return dict(c, name=name, **kw) if name else dict(c, **kw)


def _attend(name: str, **kw: Any) -> Dict[str, Any]:
    c = dict(kind="attend", batch=1, q_lo=1, q_hi=1, len_lo=1, len_hi=1, prefix=0, page=16, hq=32, hkv=4, dim=128,
             dtype="f16", lse=False)
    return dict(c, name=name, **kw) if name else dict(c, **kw)


def _sample(name: str, **kw: Any) -> Dict[str, Any]:
    c = dict(kind="sample", rows=1, vocab=151936, dtype="f32", temperature=0.8, top_k=0, top_p=1.0, min_p=0.0,
             per_row=False)
    return dict(c, name=name, **kw) if name else dict(c, **kw)


def listed() -> List[Dict[str, Any]]:
    return [
        # One user's decode step far into a conversation: fp32 projections, per-head norms.
        _append("append_decode_1", len_lo=30011, len_hi=30011, norm=True, src="f32"),
        # A batch of 64 users decoding behind a shared system prompt.
        _append("append_decode_64", batch=64, len_lo=20, len_hi=900, prefix=8192, norm=True, src="f32", dtype="bf16"),
        # Seven prompts of uneven lengths prefilled together, interleaved rotation of half the head.
        _append("append_prompts", batch=7, q_lo=90, q_hi=1111, len_lo=90, len_hi=1111, prefix=1000, page=64, hkv=8,
                rot=64, interleaved=True),
        # One user's decode step: 5003 cached keys, no shared prefix.
        _attend("attend_decode_1", len_lo=5003, len_hi=5003),
        # 64 users behind one system prompt, a few hundred keys of their own.
        _attend("attend_decode_64", batch=64, len_lo=20, len_hi=900, prefix=8192),
        # A large serving batch behind a long shared document.
        _attend("attend_decode_256", batch=256, len_lo=1, len_hi=600, prefix=16000, dtype="bf16", page=32),
        # 32 long conversations of uneven lengths without a prefix: the cache stream itself.
        _attend("attend_long_32", batch=32, len_lo=1500, len_hi=16001, hkv=8, page=64),
        # Speculative verification: 16 sequences of up to 6 draft tokens, a prefix that ends inside a page.
        _attend("attend_verify_16", batch=16, q_lo=2, q_hi=6, len_lo=30, len_hi=2000, prefix=3001, dim=64, hq=16, hkv=8,
                lse=True),
        # Prompts prefilled against a shared prefix in one call.
        _attend("attend_prompts", batch=6, q_lo=200, q_hi=1201, len_lo=200, len_hi=1201, prefix=4097, page=64, hkv=8,
                dtype="bf16"),
        # One user's next token from the output head's fp32 logits.
        _sample("sample_1", top_k=40, top_p=0.95),
        # A serving batch whose rows ask for different settings, greedy ones among them.
        _sample("sample_48_mixed", rows=48, per_row=True, top_k=200, top_p=0.9, min_p=0.02, dtype="f16"),
        # A large batch drawn from the whole distribution but its far tail.
        _sample("sample_256", rows=256, vocab=131072, temperature=1.1, top_p=0.98),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random) -> Dict[str, Any]:
    kind = rng.choice(("append", "attend", "attend", "sample"))
    if kind == "sample":
        vocab = _log(rng, 300, 200000)
        rows = _log(rng, 1, max(1, min(256, 30000000 // vocab)))
        return _sample("", rows=rows, vocab=vocab, dtype=rng.choice(("f32", "f16", "bf16")),
                       temperature=round(rng.uniform(0.3, 1.5), 2), top_k=rng.choice((0, 0, _log(rng, 1, 2000))),
                       top_p=rng.choice((1.0, round(rng.uniform(0.3, 0.99), 3))),
                       min_p=rng.choice((0.0, round(rng.uniform(0.001, 0.2), 3))), per_row=rng.random() < 0.3)
    hkv = rng.choice((1, 2, 4, 8))
    dim = rng.choice((64, 128, 128, 256))
    hq = hkv * rng.choice((1, 2, 4, 5, 8))
    c = dict(page=rng.choice((16, 32, 64, 128)), hkv=hkv, dim=dim, hq=hq, dtype=rng.choice(("f16", "bf16")))
    shape = rng.choice(("decode", "decode", "verify", "prompts"))
    if shape == "prompts":
        q = _log(rng, 20, 900)
        c.update(batch=rng.randint(1, 6), q_lo=max(1, q // 4), q_hi=q)
    else:
        c.update(batch=_log(rng, 1, 128), q_lo=1, q_hi=1 if shape == "decode" else rng.randint(2, 8))
    most = 16000 if c["batch"] <= 32 else 2000
    hi = c["q_hi"] + _log(rng, 1, most if shape != "prompts" else 1000)
    c.update(len_lo=rng.randint(c["q_hi"], hi), len_hi=hi, prefix=rng.choice((0, _log(rng, 10, 12000))))
    if kind == "append":
        c["len_hi"] = c["len_lo"] = min(c["len_hi"], 2000 + c["q_hi"])
        return _append("", rot=rng.choice((dim, dim // 2)), interleaved=rng.random() < 0.4, norm=rng.random() < 0.5,
                       src=rng.choice(("f32", "f16", "bf16")), **c)
    return _attend("", lse=rng.random() < 0.3, **c)


def _spread(lo: int, hi: int, n: int, salt: int) -> List[int]:
    """n lengths from lo to hi, both among them where n > 1, in an order of their own."""
    v = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]
    random.Random(salt).shuffle(v)
    return v


def _lengths(c: Dict[str, Any]):
    """(queries, own keys) of each sequence: a sequence holds its queries' keys at least."""
    q = _spread(c["q_lo"], c["q_hi"], c["batch"], 1)
    if c["len_lo"] == c["q_lo"] and c["len_hi"] == c["q_hi"]:
        return q, list(q)  # prompts: every key is one of this call's tokens
    return q, [max(a, b) for a, b in zip(q, _spread(c["len_lo"], c["len_hi"], c["batch"], 2))]


def work(c: Dict[str, Any]) -> Dict[str, float]:
    if c["kind"] == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": float(n * _BYTES[c["dtype"]] + 16 * c["rows"]), "flops": 20.0 * n}
    q, lens = _lengths(c)
    T, row = sum(q), c["dim"] * _BYTES[c["dtype"]]
    if c["kind"] == "append":
        n = T * (c["hq"] + 2 * c["hkv"]) * c["dim"]
        return {"bytes": float(n * (_BYTES[c["src"]] + _BYTES[c["dtype"]])), "flops": 6.0 * n}
    keys = c["prefix"] + sum(lens)
    seen = sum(a * c["prefix"] + a * (b - a) + a * (a + 1) // 2 for a, b in zip(q, lens))
    return {"bytes": float(2 * T * c["hq"] * row + 2 * keys * c["hkv"] * row), "flops": 4.0 * c["hq"] * c["dim"] * seen}


# ------------------------------------------------------------------ inputs
def prepare(c: Dict[str, Any], seed: int) -> Dict[str, Any]:
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape: int) -> torch.Tensor:
        return torch.randn(*shape, generator=g, device="cuda")

    if c["kind"] == "sample":
        B, V = c["rows"], c["vocab"]
        # a head's logits: a wide bell with a few tokens well above it
        x = normal(B, V) * 2.0
        top = torch.randint(0, V, (B, min(V, 30)), generator=g, device="cuda")
        x.scatter_add_(1, top, torch.rand(top.shape, generator=g, device="cuda") * 12.0)
        s = dict(c, logits=x.to(_TYPES[c["dtype"]]), u=torch.rand(B, generator=g, device="cuda"))
        if c["per_row"]:  # each row its own settings: some greedy, some without one filter or the other
            def pick(v: torch.Tensor, off: float, every: int, at: int) -> torch.Tensor:
                return torch.where(torch.arange(B, device="cuda") % every == at, torch.full_like(v, off), v)

            r = torch.rand(4, B, generator=g, device="cuda")
            s["temperature"] = pick(0.3 + r[0], 0.0, 7, 3)
            s["top_k"] = pick(1 + (r[1] * c["top_k"]).floor(), 0, 3, 1).to(torch.int32)
            s["top_p"] = pick(c["top_p"] + (1 - c["top_p"]) * 0.9 * r[2], 1.0, 4, 2)
            s["min_p"] = pick(c["min_p"] * r[3], 0.0, 2, 1)
        return s
    q, lens = _lengths(c)
    T, B, D, ps = sum(q), c["batch"], c["dim"], c["page"]
    dt = _TYPES[c["dtype"]]
    pages = [-(-n // ps) for n in lens]
    shared = -(-c["prefix"] // ps)
    n_pages = sum(pages) + shared + 3
    order = torch.randperm(n_pages, generator=g, device="cuda", dtype=torch.int32)
    table = torch.zeros(B, max(pages), dtype=torch.int32, device="cuda")
    fill = torch.arange(max(pages), device="cuda")[None, :] < torch.tensor(pages, device="cuda")[:, None]
    table[fill] = order[shared:shared + sum(pages)]
    s = dict(c, T=T, longest=max(lens), q_max=max(q), table=table, prefix_pages=order[:shared].clone(),
             lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
             q_start=torch.tensor([sum(q[:i]) for i in range(B + 1)], dtype=torch.int32, device="cuda"),
             k=normal(n_pages, c["hkv"], ps, D).to(dt), v=normal(n_pages, c["hkv"], ps, D).to(dt))
    ragged = c["q_hi"] > 1
    if c["kind"] == "append":
        # one fused projection's output, split into heads by views
        cat = normal(T, (c["hq"] + 2 * c["hkv"]) * D).to(_TYPES[c["src"]]) * 1.5
        parts = cat.split([c["hq"] * D, c["hkv"] * D, c["hkv"] * D], dim=1)
        s["new"] = [p.unflatten(1, (-1, D)) for p in parts]
        s["norms"] = [1 + 0.2 * normal(D), 1 + 0.2 * normal(D)] if c["norm"] else [None, None]
        s["inv_freq"] = 1e6 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])
    else:
        s["q"] = normal(T, c["hq"], D).to(dt)
    if own:  # the handles a program keeps over its steps
        p = _pkg()
        s["cache"] = p.HipPagedKVCache.from_tensors(s["k"], s["v"])
        s["steps"] = p.KVBatch(table, s["lens"], q_start=s["q_start"] if ragged else None,
                               prefix_pages=s["prefix_pages"] if shared else None, prefix_len=c["prefix"])
        if c["kind"] == "append":
            s["rope"] = p.HipRotary(D, inv_freq=s["inv_freq"], interleaved=c["interleaved"])
    return s


# ------------------------------------------------------------------ the operators
def run(s: Dict[str, Any]) -> Any:
    if own:
        if s["kind"] == "append":
            qn, kn = s["norms"]
            q = s["cache"].append(*s["new"], s["steps"], s["rope"], q_norm=qn, k_norm=kn)
            return {"q": q, "k": s["k"], "v": s["v"]}
        if s["kind"] == "attend":
            r = s["cache"].attend(s["q"], s["steps"], return_lse=s["lse"])
            return {"out": r[0], "lse": r[1]} if s["lse"] else {"out": r}
        tok, logp = _pkg().sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                         top_p=s["top_p"], min_p=s["min_p"])
        return {"token": tok, "logprob": logp}
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[s["kind"]](s)


def _token_places(s: Dict[str, Any]):
    """(sequence, own index) of every token."""
    t = torch.arange(s["T"], device="cuda")
    b = torch.searchsorted(s["q_start"], t, right=True, out_int32=False) - 1
    return b, (s["lens"][b] - s["q_start"][b + 1] + t.to(torch.int32)).long()


def _plain_append(s: Dict[str, Any]) -> Dict[str, torch.Tensor]:
    b, j = _token_places(s)
    half, dt = s["rot"] // 2, s["k"].dtype
    a = (s["prefix"] + j).double()[:, None] * s["inv_freq"]
    cos, sin = a.cos().float()[:, None, :], a.sin().float()[:, None, :]

    def norm(x: torch.Tensor, w: Any) -> torch.Tensor:
        x = x.float()
        return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w

    def turn(x: torch.Tensor) -> torch.Tensor:
        r, rest = x[..., :2 * half], x[..., 2 * half:]
        p, q = (r[..., 0::2], r[..., 1::2]) if s["interleaved"] else (r[..., :half], r[..., half:])
        p, q = p * cos - q * sin, q * cos + p * sin
        r = torch.stack((p, q), -1).flatten(-2) if s["interleaved"] else torch.cat((p, q), -1)
        return torch.cat((r, rest), -1).to(dt)

    q, k, v = s["new"]
    page, off = s["table"][b, j // s["page"]].long(), j % s["page"]
    s["k"][page, :, off] = turn(norm(k, s["norms"][1]))
    s["v"][page, :, off] = v.to(dt)
    return {"q": turn(norm(q, s["norms"][0])), "k": s["k"], "v": s["v"]}


def _gather(cache: torch.Tensor, pages: torch.Tensor, n: int) -> torch.Tensor:
    """The first n rows of the given pages [..., pages] as fp32 [..., heads, n, dim]."""
    x = cache[pages.long()].float().transpose(-4, -3)  # [..., heads, pages, page, dim]
    return x.flatten(-3, -2)[..., :n, :]


def _plain_attend(s: Dict[str, Any]) -> Dict[str, torch.Tensor]:
    T, B, H, G, D, Q = s["T"], s["batch"], s["hkv"], s["hq"] // s["hkv"], s["dim"], s["q_max"]
    b, j = _token_places(s)
    i = torch.arange(T, device="cuda") - s["q_start"][b]
    q = s["q"].float().reshape(T, H, G, D) * D ** -0.5
    # own keys: every sequence's queries padded to Q, its keys to the longest
    qp = q.new_zeros(B, Q, H, G, D)
    qp[b, i] = q
    qp = qp.permute(0, 2, 1, 3, 4).reshape(B, H, Q * G, D)
    k, v = _gather(s["k"], s["table"], s["longest"]), _gather(s["v"], s["table"], s["longest"])
    key = torch.arange(s["longest"], device="cuda")
    k, v = (x.masked_fill((key >= s["lens"][:, None])[:, None, :, None], 0.0) for x in (k, v))
    x = torch.matmul(qp, k.transpose(-1, -2)).view(B, H, Q, G, -1)
    last = torch.full((B, Q), -1, dtype=torch.long, device="cuda")
    last[b, i] = j
    x = x.masked_fill((key > last[:, :, None])[:, None, :, None, :], -math.inf)
    m = x.amax(-1)[b, :, i].reshape(T, H, G)
    if s["prefix"]:
        kp, vp = _gather(s["k"], s["prefix_pages"], s["prefix"]), _gather(s["v"], s["prefix_pages"], s["prefix"])
        xp = torch.matmul(q.permute(1, 0, 2, 3).reshape(H, T * G, D), kp.transpose(-1, -2))
        m = torch.maximum(m, xp.amax(-1).view(H, T, G).transpose(0, 1))
    mp = m.new_zeros(B, Q, H, G)
    mp[b, i] = m
    w = torch.exp(x - mp.transpose(1, 2)[..., None])
    o = torch.matmul(w.view(B, H, Q * G, -1), v).view(B, H, Q, G, D)[b, :, i]
    n = w.sum(-1)[b, :, i]
    if s["prefix"]:
        wp = torch.exp(xp - m.transpose(0, 1).reshape(H, T * G, 1))
        o = o + torch.matmul(wp, vp).view(H, T, G, D).transpose(0, 1)
        n = n + wp.sum(-1).view(H, T, G).transpose(0, 1)
    out = {"out": (o / n[..., None]).reshape(T, H * G, D).to(s["q"].dtype)}
    return dict(out, lse=(m + n.log()).reshape(T, H * G)) if s["lse"] else out


def _plain_sample(s: Dict[str, Any]) -> Dict[str, torch.Tensor]:
    x = s["logits"].double()
    B, V = x.shape

    def col(v: Any) -> torch.Tensor:
        return v.double()[:, None] if torch.is_tensor(v) else torch.full((B, 1), float(v), dtype=torch.float64, device="cuda")

    temp, k, p, least = (col(s[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    greedy = temp <= 0
    w = torch.exp((x - x.amax(1, keepdim=True)) / torch.where(greedy, torch.ones_like(temp), temp))
    sx, order = torch.sort(x, dim=1, descending=True, stable=True)  # ties by the lower index
    sw = w.gather(1, order)
    cum = sw.cumsum(1)
    rank = torch.arange(V, device="cuda")[None, :]
    keep = (rank < torch.where(k > 0, k, torch.full_like(k, V))) & (sw >= least)
    keep &= (cum - sw < p * cum[:, -1:]) | (p >= 1)
    keep = torch.where(greedy, rank == 0, keep)
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, sw, torch.zeros_like(sw)))
    c = kept.cumsum(1)
    tok = (c <= s["u"].double()[:, None] * c[:, -1:]).sum(1)
    tok = torch.minimum(tok, (kept > 0).long().mul(torch.arange(V, device="cuda")).amax(1))
    return {"token": tok, "logprob": (kept.gather(1, tok[:, None]) / c[:, -1:]).log().squeeze(1).float()}


# ------------------------------------------------------------------ float64, from the definitions
def exact(c: Dict[str, Any], seed: int) -> Any:
    s = prepare(c, seed)
    if c["kind"] == "append":
        return _exact_append(s)
    return _exact_attend(s) if c["kind"] == "attend" else _exact_sample(s)


def _exact_append(s: Dict[str, Any]) -> Dict[str, torch.Tensor]:
    """Rotation as a product of complex numbers, sequence by sequence."""
    q_start, lens = s["q_start"].tolist(), s["lens"].tolist()
    kc, vc, table = s["k"].double(), s["v"].double(), s["table"].long()
    rot, out = s["rot"], []

    def turned(x: torch.Tensor, w: Any, z: torch.Tensor) -> torch.Tensor:
        x = x.double()
        if w is not None:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        r = x[..., :rot]
        pair = r.unflatten(-1, (-1, 2)) if s["interleaved"] else r.unflatten(-1, (2, -1)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z[:, None, :])
        y = y.flatten(-2) if s["interleaved"] else y.transpose(-1, -2).flatten(-2)
        return torch.cat((y, x[..., rot:]), -1)

    for b in range(s["batch"]):
        lo, hi = q_start[b], q_start[b + 1]
        own_at = torch.arange(lens[b] - (hi - lo), lens[b], device="cuda")
        angle = (own_at + s["prefix"]).double()[:, None] * s["inv_freq"]
        z = torch.polar(torch.ones_like(angle), angle)
        q, k, v = (x[lo:hi] for x in s["new"])
        out.append(turned(q, s["norms"][0], z))
        pg, at = table[b][own_at // s["page"]], own_at % s["page"]
        kc[pg, :, at] = turned(k, s["norms"][1], z)
        vc[pg, :, at] = v.double()
    return {"q": torch.cat(out), "k": kc, "v": vc}


def _exact_attend(s: Dict[str, Any]) -> Dict[str, torch.Tensor]:
    """One KV head of one sequence at a time: softmax of a dense masked score matrix."""
    q_start, lens, P, ps = s["q_start"].tolist(), s["lens"].tolist(), s["prefix"], s["page"]
    T, H, G, D = s["T"], s["hkv"], s["hq"] // s["hkv"], s["dim"]
    out = torch.empty(T, H * G, D, dtype=torch.float64, device="cuda")
    lse = torch.empty(T, H * G, dtype=torch.float64, device="cuda")
    for b in range(s["batch"]):
        lo, hi, n = q_start[b], q_start[b + 1], lens[b]
        pages = torch.cat((s["prefix_pages"], s["table"][b, :-(-n // ps)])).long()
        held = -(-P // ps) * ps
        rows = torch.cat((torch.arange(P), torch.arange(held, held + n))).to("cuda")
        late = torch.arange(n, device="cuda")[None, :] > torch.arange(n - (hi - lo), n, device="cuda")[:, None]
        late = torch.cat((late.new_zeros(hi - lo, P), late), 1)
        for h in range(H):
            k = s["k"][pages, h].reshape(-1, D)[rows].double()
            v = s["v"][pages, h].reshape(-1, D)[rows].double()
            x = s["q"][lo:hi, h * G:(h + 1) * G].double() @ k.T / math.sqrt(D)
            x = torch.where(late[:, None, :], -math.inf, x)
            lse[lo:hi, h * G:(h + 1) * G] = torch.logsumexp(x, -1)
            out[lo:hi, h * G:(h + 1) * G] = torch.softmax(x, -1) @ v
    return {"out": out, "lse": lse} if s["lse"] else {"out": out}


def _exact_sample(s: Dict[str, Any]) -> Dict[str, Any]:
    """numpy, row by row; the tokens are whole numbers and have no float64 value."""
    x, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    par = {n: s[n].double().cpu().numpy() if torch.is_tensor(s[n]) else np.full(len(u), float(s[n]))
           for n in ("temperature", "top_k", "top_p", "min_p")}
    logp = np.zeros(len(u))
    for r, row in enumerate(x):
        if par["temperature"][r] <= 0:
            continue
        e = np.exp((row - row.max()) / par["temperature"][r])
        prob = e / e.sum()
        order = np.lexsort((np.arange(len(row)), -row))
        n = len(row)
        if par["top_k"][r] > 0:
            n = min(n, int(par["top_k"][r]))
        if par["top_p"][r] < 1:
            n = min(n, 1 + int(np.searchsorted(np.cumsum(prob[order]), par["top_p"][r])))
        n = max(1, min(n, int((e >= par["min_p"][r]).sum())))
        kept = np.sort(order[:n])
        c = np.cumsum(e[kept])
        at = min(int(np.searchsorted(c, u[r] * c[-1], side="right")), n - 1)
        logp[r] = math.log(e[kept[at]] / c[-1])
    return {"token": None, "logprob": torch.from_numpy(logp)}
