"""sample_tokens where far tokens have no weight: w is held in multiples of 2^-s of the largest, s =
min(51, 62 - ceil(log2 V)), and a token of less than half of one is not drawn, not even at u = 0, in
whichever part of a long row it lies and however many of its kind lie there."""

import math

import pytest

from gpu_helpers import log
from kv_helpers import DTYPES

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda", 0)


# vocabulary, logit of the tokens without weight: half of 2^-s is e^-33.96 for 2^14 tokens, e^-29.81 for 2^20,
# e^-31.88 for 131072 (s = 45), e^-36.04 for 2048 and fewer
ROWS = [(2048, -37.0), (16384, -35.0), (16384, -34.5), (40000, -34.0), (131072, -32.5), (131072, -40.0), (1 << 20, -30.5),
        (1 << 20, -31.0)]
FILTERS = [dict(), dict(top_k=-1), dict(top_p=1 - 1e-12), dict(min_p=1e-300), dict(top_k=-1, top_p=1 - 1e-12, min_p=1e-300)]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("i", range(len(FILTERS)))
@pytest.mark.parametrize("vocab,far", ROWS)
def test_far_tokens_are_not_drawn_at_u_0(dev, vocab, far, i, dt):
    """One token of weight 1 in the last slice, and in a second row one of weight e^-20 among the far ones of the
    first: u = 0 draws the first token that has a weight."""
    from pgmoe import sample_tokens
    log(f"sample far vocab={vocab} far={far} {FILTERS[i]} {dt}")
    s = min(51, 62 - math.ceil(math.log2(vocab)))
    x = torch.full((2, vocab), far).to(DTYPES[dt])
    far = float(x[0, 0])
    assert far < -(s + 1) * math.log(2.0) - 1e-6  # no weight, by the definition
    top, near = vocab - 700, min(8192, vocab - 800) - 100
    x[:, top] = 0.0
    x[1, near] = -20.0
    kw = {n: vocab - 1 if v == -1 else v for n, v in FILTERS[i].items()}
    tok, lp = sample_tokens(x.to(dev), torch.zeros(2, device=dev), 1.0, **kw)
    assert tok.tolist() == [top, near]
    # log w, to one step of fp32 and what the weights' fixed point can be off by: V halves of a unit
    fixed = vocab * 2.0 ** -(s + 1)
    assert abs(float(lp[0])) <= fixed + 2.0 ** -24 and abs(float(lp[1]) + 20.0 + math.log1p(math.exp(-20.0))) <= fixed + 20 * 2.0 ** -23


@pytest.mark.parametrize("vocab,far", ROWS)
def test_far_tokens_leave_the_draw_of_others(dev, vocab, far):
    """Beside far tokens the others are drawn as if those were not there."""
    from pgmoe import sample_tokens
    log(f"sample far others vocab={vocab} far={far}")
    n = 64
    g = torch.Generator().manual_seed(vocab)
    at = torch.randperm(vocab, generator=g)[:20].sort().values
    near = torch.randn(20, generator=g) * 3
    near[7] = 9.0  # the maximum; the far ones lie `far` below it
    x = torch.full((1, vocab), far + 9.0)
    x[0, at] = near
    u = (torch.arange(n) + 0.5) / n
    tok, lp = sample_tokens(x.expand(n, -1).to(dev), u.to(dev))
    w = torch.softmax(near.double(), 0)
    c = torch.cumsum(w, 0)
    want = (c[None, :] <= u[:, None].double() * c[-1]).sum(1)
    assert torch.equal(tok.cpu(), at[want])
    assert float((lp.cpu().double() - w.log()[want]).abs().max()) <= 2.0 ** -23 * 20 + vocab * 2.0 ** -40
