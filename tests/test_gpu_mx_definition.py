"""Microscaled operators against the float64 formulas where roundings on the way would show: codes next to borders, values
near the ends of fp32's range."""

import pytest

import mx_helpers as H

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FMTS = ["e4m3", "e2m1"]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda", 0)


# ---------------------------------------------------------------- norm
def _norm64(h, w, eps):
    return h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


@pytest.mark.parametrize("fmt,rows,cols,dt,ddt", [
    ("e4m3", 2000, 4096, torch.float32, torch.float16), ("e2m1", 2000, 4096, torch.float32, torch.float32),
    ("e4m3", 700, 8192, torch.bfloat16, torch.float32), ("e4m3", 3000, 1024, torch.float16, None),
    ("e4m3", 100, 20000, torch.float32, torch.bfloat16), ("e2m1", 9000, 224, torch.float32, None), ("e4m3", 500, 4064, torch.float32, None)])
def test_norm_codes_are_the_formulas(dev, fmt, rows, cols, dt, ddt):
    """Every code and scale byte of millions: nothing is rounded before them but to 64 bits."""
    from pgmoe import exec_fused_add_rmsnorm_mx, exec_fused_rmsnorm_mx
    g = torch.Generator().manual_seed(rows + cols)
    x = (3 * torch.randn(rows, cols, generator=g) * torch.exp(0.5 * torch.randn(cols, generator=g))).to(dt)
    w = 1 + 0.2 * torch.randn(cols, generator=g)
    h = x.double()
    if ddt is None:
        t = exec_fused_rmsnorm_mx(x.to(dev), w.to(dev), 1e-6, fmt)
    else:
        d = torch.randn(rows, cols, generator=g).to(ddt)
        h = h + d.double()
        got, t = exec_fused_add_rmsnorm_mx(x.to(dev), d.to(dev), w.to(dev), 1e-6, fmt)
        assert torch.equal(got.cpu(), h.float())
    codes, e = H.encode(_norm64(h, w, float(torch.tensor(1e-6))), fmt)  # eps as the C ABI takes it, in fp32
    assert torch.equal(H.scales(t), e)
    assert torch.equal(H.unpack(t), codes)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("cols", [64, 512, 2048, 4096, 8192, 16512])
def test_norm_of_far_rows(dev, fmt, cols):
    """Rows whose squares are beyond fp32's range, or below it with nothing added."""
    from pgmoe import exec_fused_add_rmsnorm_mx, exec_fused_rmsnorm_mx
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(6, cols, generator=g) * torch.tensor([1e25, 5e37, 1e-25, 1e-37, 1.0, 1e19])[:, None]
    w = 1 + 0.2 * torch.randn(cols, generator=g)
    for eps in (0.0, 1e-6):
        codes, e = H.encode(_norm64(x.double(), w, float(torch.tensor(eps))), fmt)
        t = exec_fused_rmsnorm_mx(x.to(dev), w.to(dev), eps, fmt)
        h, u = exec_fused_add_rmsnorm_mx(x.to(dev), torch.zeros_like(x).to(dev), w.to(dev), eps, fmt)
        assert torch.equal(h.cpu(), x)
        for v in (t, u):
            assert torch.equal(H.scales(v), e) and torch.equal(H.unpack(v), codes)
