"""HipPagedKVCache.append with the forms of HipRotary (given frequencies, factors, scaled positions) and with inputs
that cannot be read 16 bytes at a time."""

import math

import pytest

from gpu_helpers import log
from kv_helpers import DTYPES, HALF_STEP, Step, norm_reference, rotate_reference

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda", 0)


def _step(dim, dt, seed):
    s = Step([3, 1, 17], [40, 2000, 17], 6, 2, dim, 32, 5000, dtype=DTYPES[dt], seed=seed)
    return s, [s.randn(s.T, n, dim) * 2 for n in (6, 2, 2)]


def _positions(s):
    return torch.tensor([s.prefix + ln - m + i for m, ln in zip(s.q_lens, s.lens) for i in range(m)])


def _places(s):
    at = [(int(s.table[b, j // s.page]), j % s.page) for b, (m, ln) in enumerate(zip(s.q_lens, s.lens))
          for j in range(ln - m, ln)]
    return [torch.tensor(x) for x in zip(*at)]


def _cache(s, dev):
    from pgmoe import HipPagedKVCache
    return HipPagedKVCache(s.n_pages, s.page, s.hkv, s.dim, dtype=s.dtype, device=dev)


# freq: given as frequencies of their own; factors: rope_freqs of a file; scale of the positions; where the tensors lie
FORMS = [dict(freq=True), dict(freq=True, where="cuda"), dict(factors=True), dict(factors=True, where="cuda"),
         dict(scale=0.25), dict(scale=8.0), dict(freq=True, factors=True, scale=0.5, where="cuda")]


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dim,rot,dt", [(64, 32, "bf16"), (128, 128, "f16"), (256, 80, "f16")])
@pytest.mark.parametrize("i", range(len(FORMS)))
def test_rotary_forms_match_float64(dev, i, dim, rot, dt, inter):
    """The angle is position * scale * frequency / factor, formed in float64.  Tolerance as of the plain form: half a step
    of the result, and the angle's last rounding to fp32, cosine, sine and products: 16 roundings of 2^-24 of the
    pair's magnitudes; 2^-25: fp16 below its range."""
    from pgmoe import HipRotary
    log(f"append rotary {FORMS[i]} dim={dim} rot={rot} inter={inter}")
    f = FORMS[i]
    s, (q, k, v) = _step(dim, dt, 7 * i + dim)
    where = f.get("where", "cpu")
    inv = 1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    kw = dict(interleaved=inter)
    if f.get("freq"):
        inv = 0.9 * 5e5 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot) + 1e-7
        kw.update(inv_freq=inv.to(where))
    else:
        kw.update(base=1e4, rotary_dim=rot, device=dev)
    if f.get("factors"):
        factors = 1 + 7 * torch.rand(rot // 2, generator=s.gen)
        kw.update(freq_factors=factors.to(where))
        inv = inv / factors.double()
    kw.update(position_scale=f.get("scale", 1.0))
    rope = HipRotary(dim, **kw)
    assert rope.rotary_dim == rot and rope.device.type == "cuda"
    c = _cache(s, dev)
    got = c.append(q.to(dev), k.to(dev), v.to(dev), s.batch(dev), rope).cpu()
    pos = _positions(s).double() * f.get("scale", 1.0)
    pg, ro = _places(s)
    for y, x in ((got, q), (c.k.cpu()[pg, :, ro], k)):
        ref, mag = rotate_reference(x, pos, inv, inter)
        tol = HALF_STEP[s.dtype] * ref.abs() + 16 * 2.0 ** -24 * mag + 2.0 ** -25
        assert bool(((y.double() - ref).abs() <= tol).all()), float(((y.double() - ref).abs() - tol).max())
    assert torch.equal(c.v.cpu()[pg, :, ro], v.to(s.dtype))


def test_rotary_refusals(dev):
    from pgmoe import HipRotary
    log("rotary refusals")
    inv = torch.ones(16, dtype=torch.float64)
    for kw in (dict(inv_freq=inv, rotary_dim=64), dict(inv_freq=inv[None]), dict(inv_freq=inv[:7]), dict(inv_freq=torch.ones(80)),
               dict(freq_factors=torch.ones(31), rotary_dim=64), dict(position_scale=math.inf), dict(attn_factor=math.nan),
               dict(base=0.0), dict(base=math.nan), dict(rotary_dim=0)):
        with pytest.raises(ValueError):
            HipRotary(128, device=dev, **kw)


def _laid_out(x, how, dev):
    """x [T, H, D] on the device, its rows at odd places."""
    T, H, D = x.shape
    if how == "unaligned":
        y = torch.full((T * H * D + 1,), 9.0, dtype=x.dtype, device=dev)[1:].view(T, H, D)
    elif how == "odd token stride":
        y = torch.full((T, H * D + 3), 9.0, dtype=x.dtype, device=dev)[:, :H * D].unflatten(1, (H, D))
    elif how == "odd head stride":
        y = torch.full((T, H, D + 1), 9.0, dtype=x.dtype, device=dev)[..., :D]
    elif how == "heads first":
        y = torch.full((H, T, D), 9.0, dtype=x.dtype, device=dev).transpose(0, 1)
    elif how == "elements apart":
        y = torch.full((T, H, D, 2), 9.0, dtype=x.dtype, device=dev)[..., 0]
    elif how == "columns first":
        y = torch.full((D, H, T), 9.0, dtype=x.dtype, device=dev).permute(2, 1, 0)
    else:  # every second token of a larger tensor
        y = torch.full((2 * T, H, D), 9.0, dtype=x.dtype, device=dev)[::2]
    return y.copy_(x)


@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("how", ["unaligned", "odd token stride", "odd head stride", "heads first", "elements apart",
                                 "columns first", "every second"])
def test_append_takes_any_layout(dev, how, src):
    """The same bits as contiguous inputs give, with norms and rotation; the norm weights unaligned and in half too."""
    from pgmoe import HipRotary
    log(f"append layout {how} {src}")
    s, x = _step(128, "f16", 3)
    x = [t.to(DTYPES[src]) for t in x]
    rope = HipRotary(128, base=1e6, device=dev)
    w = (1 + 0.3 * s.randn(2, 128)).half()
    plain, odd = _cache(s, dev), _cache(s, dev)
    want = plain.append(*[t.to(dev) for t in x], s.batch(dev), rope, w[0].float().to(dev), w[1].float().to(dev))
    shifted = torch.empty(129, device=dev)[1:].copy_(w[1].float())
    given = [_laid_out(t, how, dev) for t in x]
    got = odd.append(*given, s.batch(dev), rope, w[0].to(dev), shifted)
    assert torch.equal(got, want) and torch.equal(odd.k, plain.k) and torch.equal(odd.v, plain.v)
    for t, g in zip(x, given):
        assert torch.equal(g.cpu(), t)
    # and against the definition
    pos = _positions(s)
    ref, mag = rotate_reference(norm_reference(x[0], w[0]), pos, 1e6 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128), False)
    tol = HALF_STEP[s.dtype] * ref.abs() + 32 * 2.0 ** -24 * mag + 2.0 ** -25
    assert bool(((got.cpu().double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("how", ["odd token stride", "odd head stride", "heads first", "elements apart", "columns first", "every second"])
def test_attend_takes_any_layout(dev, how):
    log(f"attend layout {how}")
    from pgmoe import HipPagedKVCache
    s, (q, _, _) = _step(128, "bf16", 5)
    k, v = s.pages()
    c = HipPagedKVCache.from_tensors(k.to(dev), v.to(dev))
    q = q.to(s.dtype)
    assert torch.equal(c.attend(_laid_out(q, how, dev), s.batch(dev)), c.attend(q.to(dev), s.batch(dev)))
