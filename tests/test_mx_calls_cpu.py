"""Microscaled calls without a GPU: arguments of later forms."""

import inspect

import pytest

from pgmoe import _lib

torch = pytest.importorskip("torch")

OK, INVALID, UNSUPPORTED = 0, -1, -2
P = 0x10000  # an aligned address that no call reaches


def test_fp32_sums_are_part_of_the_outputs_type():
    L, wide = _lib.lib(), _lib.MX_FP32_SUMS
    none, some = _lib.Mx(None, None, 128, 16, 0, 128, 8), _lib.Mx(P, P, 128, 16, 4, 128, 8)
    for dt in (0, 1, 30):
        assert L.pgmoe_mx_linear(P, 16, none, None, None, dt + wide, None) == OK
        assert L.pgmoe_mx_linear_values(P, 16, None, 0, 128, 0, 128, 8, None, None, dt + wide, None, 0, None) == OK
    for dt in (2 + wide, 8 + wide, 2 * wide, 3 * wide, 0x80 + wide, -1, -wide, wide - (1 << 31)):
        assert L.pgmoe_mx_linear(P, 16, some, None, P, dt, None) == UNSUPPORTED
        assert L.pgmoe_mx_linear_values(P, 16, P, 0, 128, 4, 128, 8, None, P, dt, None, 0, None) == UNSUPPORTED
    assert L.pgmoe_mx_dequantize(some, P, wide, None) == UNSUPPORTED
    assert L.pgmoe_mx_linear(P, 16, some, None, P + 8, wide, None) == INVALID


def test_fp32_sums_are_asked_for_by_name():
    from pgmoe import HipMXLinear
    for f in (HipMXLinear.__init__, HipMXLinear.from_gguf):
        assert inspect.signature(f).parameters["fp32_sums"].default is False
    assert "fp32_sums" in HipMXLinear.__doc__ and "2^-13" in HipMXLinear.__doc__
