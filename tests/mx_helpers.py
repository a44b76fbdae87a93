"""Float64 definitions of the microscaled blocks and their product, on the CPU."""

from __future__ import annotations

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [m / 512 for m in range(8)] + [(8 + m) / 8 * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]
LIMIT = {"e4m3": 448.0, "e2m1": 6.0}
TOP = {"e4m3": 8, "e2m1": 2}  # exponent of the format's largest power of two
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def table(fmt: str) -> torch.Tensor:
    return torch.tensor(E4M3 if fmt == "e4m3" else E2M1, dtype=torch.float64)


def exponents(top: torch.Tensor, fmt: str) -> torch.Tensor:
    """E of blocks whose largest magnitude is `top` (float64)."""
    e = torch.frexp(top).exponent.long() - 1 - TOP[fmt]
    return torch.where(top > 0, e, torch.full_like(e, -127)).clamp(min=-127)


def encode(x: torch.Tensor, fmt: str):
    """(codes one a value, E + 127) as int64 of x [rows, cols]."""
    b = x.double().reshape(x.shape[0], x.shape[1] // 32, 32)
    bad = ~torch.isfinite(b).all(-1)
    b = torch.where(bad[..., None], torch.zeros_like(b), b)
    e = exponents(b.abs().amax(-1), fmt)
    v = torch.ldexp(b, -e[..., None])
    t = table(fmt)
    a = v.abs().clamp(max=LIMIT[fmt])
    lo = torch.searchsorted(t, a.contiguous(), right=True) - 1
    hi = (lo + 1).clamp(max=len(t) - 1)
    down, up = a - t[lo], t[hi] - a
    at = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    at = at + torch.where(torch.signbit(v), 128 if fmt == "e4m3" else 8, 0)
    at = torch.where(bad[..., None], torch.zeros_like(at), at)
    e = torch.where(bad, torch.full_like(e, 128), e)
    return at.reshape(x.shape), e + 127


def unpack(t) -> torch.Tensor:
    """The codes of an MXTensor, one a value, int64 on the CPU."""
    c = t.codes.cpu().long().flatten(0, -2) if t.codes.dim() > 1 else t.codes.cpu().long()[None]
    return c if t.fmt == "e4m3" else torch.stack((c & 15, c >> 4), -1).flatten(1)


def scales(t) -> torch.Tensor:
    s = t.scales.cpu().long()
    return s.flatten(0, -2) if s.dim() > 1 else s[None]


def decode(codes: torch.Tensor, e: torch.Tensor, fmt: str) -> torch.Tensor:
    """float64 values of codes (one a value) and scale bytes."""
    half = 128 if fmt == "e4m3" else 8
    t = table(fmt)
    if fmt == "e4m3":
        t = torch.cat((t, torch.tensor([float("nan")], dtype=torch.float64)))
    v = t[codes % half] * (1.0 - 2.0 * (codes // half))
    s = torch.where(e == 255, torch.full(e.shape, float("nan"), dtype=torch.float64), torch.exp2(e.double() - 127))
    return v * s.repeat_interleave(32, 1)


def values(t) -> torch.Tensor:
    return decode(unpack(t), scales(t), t.fmt)


def pack(codes: torch.Tensor, fmt: str) -> torch.Tensor:
    c = codes.to(torch.uint8)
    return c if fmt == "e4m3" else c[..., 0::2] | c[..., 1::2] << 4


def check_blocks(t, y: torch.Tensor, rel: float) -> None:
    """t holds blocks of values that are off y (float64) by at most rel of each: E is that of a largest magnitude
    within rel of y's, a value is off by half a step of the format at that E (or held to its limit) and rel more."""
    y = y.reshape(-1, y.shape[-1])
    v, e = values(t), scales(t)
    top = y.abs().reshape(y.shape[0], -1, 32).amax(-1)
    lo, hi = exponents(top * (1 - rel), t.fmt) + 127, exponents(top * (1 + rel), t.fmt) + 127
    assert ((e >= lo) & (e <= hi)).all(), "scale bytes"
    unit = torch.exp2(e.double() - 127).repeat_interleave(32, 1)
    a = y.abs() / unit
    mant, least = (3, -6) if t.fmt == "e4m3" else (1, 0)
    step = torch.exp2((torch.frexp(a).exponent.double() - 1).clamp(min=least) - mant)
    bound = torch.maximum(0.5 * step, a * (1 + rel) - LIMIT[t.fmt]) + rel * a
    off = (v / unit - y / unit).abs()
    worst = (off / bound).max().item()
    assert worst <= 1.0 + 1e-9, f"{worst} of the bound"


def product(x: torch.Tensor, w: torch.Tensor, bias=None):
    """(y, what bounds its error) in float64 of values x [M, K], w [N, K]: the sum of the products' magnitudes and the
    sum over eight neighbours each of (largest x) (largest w), at least their largest product."""
    y, s = x @ w.T, x.abs() @ w.abs().T
    near = x.abs().unflatten(1, (-1, 8)).amax(-1) @ w.abs().unflatten(1, (-1, 8)).amax(-1).T
    return (y, (s, near)) if bias is None else (y + bias.double().cpu(), (s + bias.double().cpu().abs(), near))


def check_product(got: torch.Tensor, y: torch.Tensor, s, K: int, cut: bool = False) -> None:
    """A sum over K in fp32, up to 128 products at a time onto a running sum, then of up to 16 parts: each of the
    K / 128 + 17 additions is off by at most 2^-21 of the magnitudes' sum (products are aligned to the largest of eight and
    cut at 2^-24 of it: 8 of them in each of 16 such sums, and the sums' own additions); then one rounding.
    cut (16-bit outputs of 8-bit activations): the instruction cuts the products of eight neighbours at 2^-13 of the
    largest one's power of two, each by less than that: 8 2^-13 of the largest for each eight."""
    s, near = s
    got64 = got.double().cpu().reshape(y.shape)
    bad = ~torch.isfinite(y)
    assert torch.equal(torch.isnan(got64), bad), "NaN in other places"
    half = HALF_STEP[got.dtype]
    bound = (K / 128 + 17) * 2.0 ** -21 * s + half * y.abs() + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    if cut:
        assert got.dtype != torch.float32
        bound = bound + 2.0 ** -10 * near * (1 + half)
    off = (got64 - y).abs()
    worst = torch.where(bad | (s == 0), torch.zeros_like(off), off / bound).max().item()
    assert worst <= 1.0, f"{worst} of the bound"
    assert (got64[(s == 0) & ~bad] == 0).all()
