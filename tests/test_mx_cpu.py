"""Microscaled blocks without a GPU: what the C ABI and the Python surface refuse, sizes, and the tests' own oracle."""

import pytest

import mx_helpers as H
from pgmoe import _lib

torch = pytest.importorskip("torch")

OK, INVALID, UNSUPPORTED = 0, -1, -2
P = 0x10000  # an aligned address that no call reaches


def _blocks(fmt=8, rows=4, cols=128, codes=P, scales=P, code_stride=None, scale_stride=None):
    return _lib.Mx(codes, scales, cols if code_stride is None else code_stride, 16 if scale_stride is None else scale_stride,
                   rows, cols, fmt)


BAD_BLOCKS = [
    (dict(fmt=6), UNSUPPORTED), (dict(rows=-1), INVALID), (dict(rows=1 << 24), INVALID), (dict(cols=0), INVALID),
    (dict(cols=48, code_stride=48), INVALID), (dict(cols=(1 << 22) + 32, code_stride=1 << 23), INVALID), (dict(code_stride=112), INVALID),
    (dict(code_stride=136), INVALID), (dict(scale_stride=3), INVALID), (dict(scale_stride=20), INVALID), (dict(scale_stride=1 << 24), INVALID),
    (dict(codes=None), INVALID), (dict(scales=None), INVALID), (dict(codes=P + 8), INVALID), (dict(scales=P + 4), INVALID),
    (dict(code_stride=1 << 40), INVALID), (dict(code_stride=(1 << 23) + 16), INVALID)]


@pytest.mark.parametrize("kw,rc", BAD_BLOCKS)
def test_blocks_are_checked_at_every_entry(kw, rc):
    L, t = _lib.lib(), _blocks(**kw)
    assert L.pgmoe_mx_quantize(P, 0, 128, t, None) == rc
    assert L.pgmoe_mx_dequantize(t, P, 0, None) == rc
    assert L.pgmoe_add_rmsnorm_mx(P, 0, None, 0, P, 1e-6, None, t, None) == rc
    assert L.pgmoe_mx_act_mul(P, 128, P, 128, 0, 0, t, None) == rc
    assert L.pgmoe_mx_linear(P, 16, t, None, P, 0, None) == rc
    assert L.pgmoe_mx_quantize(P, 0, 128, None, None) == INVALID
    assert L.pgmoe_mx_pack(t, P, None) in (rc, UNSUPPORTED)


def test_no_rows_are_no_work():
    L, t = _lib.lib(), _blocks(rows=0, codes=None, scales=None)
    assert L.pgmoe_mx_quantize(None, 0, 128, t, None) == OK
    assert L.pgmoe_mx_dequantize(t, None, 0, None) == OK
    assert L.pgmoe_add_rmsnorm_mx(None, 0, None, 0, None, 1e-6, None, t, None) == OK
    assert L.pgmoe_mx_act_mul(None, 128, None, 128, 0, 0, t, None) == OK
    assert L.pgmoe_mx_linear(None, 16, t, None, None, 0, None) == OK


def test_other_arguments_are_checked():
    L, t = _lib.lib(), _blocks()
    for p, dt, stride, rc in [(None, 0, 128, INVALID), (P + 4, 0, 128, INVALID), (P, 5, 128, UNSUPPORTED), (P, 0, 120, INVALID),
                              (P, 0, 130, INVALID), (P, 1, 132, INVALID), (P, 1, 1 << 40, INVALID)]:
        assert L.pgmoe_mx_quantize(p, dt, stride, t, None) == rc
        assert L.pgmoe_mx_act_mul(p, stride, P, 128, dt, 0, t, None) == rc
        assert L.pgmoe_mx_act_mul(P, 128, p, stride, dt, 0, t, None) == rc
    assert L.pgmoe_mx_act_mul(P, 128, P, 128, 0, 2, t, None) == UNSUPPORTED
    assert L.pgmoe_mx_dequantize(t, None, 0, None) == INVALID
    assert L.pgmoe_mx_dequantize(t, P, 2, None) == UNSUPPORTED
    norm = lambda **k: L.pgmoe_add_rmsnorm_mx(*dict(dict(x=P, dt=0, d=P, ddt=0, w=P, eps=1e-6, h=P), **k).values(), t, None)  # noqa: E731
    assert norm(eps=-1.0) == INVALID and norm(eps=float("nan")) == INVALID
    assert norm(x=None) == INVALID and norm(w=None) == INVALID and norm(w=P + 4) == INVALID and norm(h=P + 8) == INVALID
    assert norm(dt=2) == UNSUPPORTED and norm(ddt=2) == UNSUPPORTED and norm(d=P + 8) == INVALID
    for out in (0, -5, 1 << 24):
        assert L.pgmoe_mx_linear(P, out, t, None, P, 0, None) == INVALID
    assert L.pgmoe_mx_linear(None, 16, t, None, P, 0, None) == INVALID
    assert L.pgmoe_mx_linear(P, 16, t, None, P + 8, 0, None) == INVALID
    assert L.pgmoe_mx_linear(P, 16, t, P + 2, P, 0, None) == INVALID
    assert L.pgmoe_mx_linear(P, 16, t, None, P, 8, None) == UNSUPPORTED
    assert L.pgmoe_mx_linear(P, (1 << 24) - 1, _blocks(rows=(1 << 24) - 1), None, P, 0, None) == UNSUPPORTED
    assert L.pgmoe_mx_pack(t, P, None) == UNSUPPORTED  # weights are e2m1
    assert L.pgmoe_mx_pack(_blocks(fmt=4, code_stride=64), None, None) == INVALID
    assert L.pgmoe_mx_pack(_blocks(fmt=4, code_stride=64, rows=0), P, None) == INVALID


def test_products_of_values():
    """Their arguments, and the workspace of the blocks of more than 16 rows."""
    L = _lib.lib()
    f = L.pgmoe_mx_linear_values_workspace_bytes
    assert f(16, 4096, 8) == f(0, 4096, 8) == 0 and f(17, 4096, 8) == 17 * (4096 + 128) and f(100, 96, 4) == 100 * (48 + 16)
    args = dict(w=P, n=16, x=P, dt=0, stride=128, rows=4, cols=128, fmt=8, bias=None, out=P, odt=0, ws=None, bytes=0)
    call = lambda **k: L.pgmoe_mx_linear_values(*dict(args, **k).values(), None)  # noqa: E731
    assert call(rows=0, x=None, w=None, out=None) == OK
    for k, rc in [(dict(x=None), INVALID), (dict(x=P + 8), INVALID), (dict(w=None), INVALID), (dict(out=None), INVALID),
                  (dict(dt=7), UNSUPPORTED), (dict(odt=7), UNSUPPORTED), (dict(fmt=5), UNSUPPORTED), (dict(cols=100), INVALID),
                  (dict(rows=-1), INVALID), (dict(rows=1 << 24), -3), (dict(stride=64), INVALID), (dict(stride=129), INVALID),
                  (dict(n=0), INVALID), (dict(rows=17), -3), (dict(rows=17, ws=P, bytes=17 * 144 - 1), -3),
                  (dict(rows=17, ws=P + 8, bytes=1 << 20), -3), (dict(bias=P + 1), INVALID)]:
        assert call(**k) == rc, k


def test_packed_bytes():
    """16-row groups of 512-input quads: 4 KB of codes and 256 bytes of scales each."""
    f = _lib.lib().pgmoe_mx_packed_bytes
    assert f(16, 512) == 4352 and f(1, 32) == 4352 and f(17, 512) == 2 * 4352 and f(16, 544) == 2 * 4352
    assert f(24576, 4096) == 24576 * 4096 * 17 // 32
    assert f(0, 512) == f(16, 0) == f(16, 48) == f(-1, 32) == f(1 << 24, 1 << 20) == -1


def test_there_is_no_cpu_path():
    from pgmoe import HipMXLinear, MXTensor, exec_fused_act_mul_mx, exec_fused_add_rmsnorm_mx, exec_fused_rmsnorm_mx, mx_quantize
    x = torch.zeros(2, 64)
    for call in (lambda: mx_quantize(x), lambda: exec_fused_rmsnorm_mx(x, torch.ones(64)),
                 lambda: exec_fused_add_rmsnorm_mx(x, x, torch.ones(64)), lambda: exec_fused_act_mul_mx(x, x),
                 lambda: MXTensor(torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)),
                 lambda: HipMXLinear.from_gguf(None, "w", device="cpu")):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_the_oracle(fmt):
    """Every code reads back as itself; a value between two codes goes to the nearer, the even one of two as near."""
    n = 127 if fmt == "e4m3" else 8
    t = H.table(fmt)
    x = torch.full((n, 32), H.LIMIT[fmt], dtype=torch.float64)  # which keeps the block's power of two at 1
    x[:, 5], x[:, 9] = t, -t
    c, e = H.encode(x, fmt)
    assert torch.equal(H.decode(c, e, fmt), x)
    mid = (t[:-1] + t[1:]) / 2
    x = torch.full((len(mid), 32), H.LIMIT[fmt], dtype=torch.float64)
    x[:, 0], x[:, 1], x[:, 2] = mid, mid * (1 + 1e-12), mid * (1 - 1e-12)
    c, e = H.encode(x, fmt)
    k = torch.arange(len(mid))
    assert torch.equal(c[:, 0], k + k % 2) and torch.equal(c[:, 1], k + 1) and torch.equal(c[:, 2], k)
    assert torch.isnan(H.decode(torch.zeros(1, 32, dtype=torch.long), torch.tensor([[255]]), fmt)).all()
