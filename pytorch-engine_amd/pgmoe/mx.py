"""Microscaled blocks: 8-bit activations and 4-bit weights in blocks of 32 that share a power of two.

    h, x = exec_fused_add_rmsnorm_mx(x, delta, norm_weight)        # the block's input, as 8-bit blocks
    gu = gate_up(x, out_dtype=torch.float16)                       # HipMXLinear on 4-bit weights
    a = exec_fused_act_mul_mx(gu[:, :I], gu[:, I:])                # silu(gate) * up, as 8-bit blocks
    delta = down(a, out_dtype=torch.float32)

A block of 32 values along a row is held as 2^E (a byte, E + 127) and codes: e4m3 (a byte each) or e2m1 (4 bits):
E = max(-127, floor(log2 max|x|) - e), e = 8 (e4m3) or 2 (e2m1); codes x / 2^E to the nearest, ties to even, at
most 448 or 6 in size.  Byte 255 makes a block NaN; blocks that hold an infinity or NaN become such ones.
e2m1 is what GGUF files hold as MXFP4 (ggml type 39): HipMXLinear.from_gguf keeps those values exactly, where
GGUFQuantLinear re-quantises them as the reference does (pygguf_engine/quant_kernels.py:906-942).

Products run on the matrix cores' own scaled form: blocks are multiplied by their powers of two in the product.
Nothing synchronises with the host but the layers' constructors.  There is no CPU path.
"""

from __future__ import annotations

import ctypes
from typing import Any, Optional, Sequence, Tuple, Union

import numpy as np
import torch
import torch.nn as nn

from ._lib import ACT_GELU_TANH, ACT_SILU, BF16, F16, F32, MX_FP32_SUMS, MXFP4, Mx, lib
from .attention import launch
from .moe import _load_lock, load_float_tensor

_DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_FMT = {"e4m3": 8, "e2m1": 4}  # bits a value
_ACT = {"silu": ACT_SILU, "gelu": ACT_GELU_TANH}
_ROWS, _COLS = 1 << 24, 1 << 22  # rows below, columns up to
_STRIDE = 1 << 23  # bytes from row to row of blocks
_FLOAT_STRIDE = 1 << 31  # elements from row to row of values


def _bits(fmt: str) -> int:
    bits = _FMT.get(fmt)
    if bits is None:
        raise NotImplementedError(f"block format {fmt!r} (e4m3 or e2m1)")
    return bits


def _row_stride(t: torch.Tensor) -> int:
    """Elements from one row of t [..., n] to the next as one matrix of rows; -1 if there is no such number."""
    if t.numel() == 0:
        return t.shape[-1]
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        return -1
    step, rows = None, 1  # innermost first; an axis of one has no stride of its own
    for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if step is None:
            step = s
        elif s != step * rows:
            return -1
        rows *= n
    return t.shape[-1] if step is None else step


def _placed(t: torch.Tensor, n: int, size: int, most: int) -> Tuple[torch.Tensor, int, int]:
    """t [..., n] of `size` bytes an element, or a contiguous copy, with rows that begin at multiples of 16 bytes, do not
    overlap and lie at most `most` elements from each other; the elements from row to row; its address."""
    s = n if t.is_contiguous() else _row_stride(t)
    p = t.data_ptr()
    if s < n or (s * size | p) & 15 or s > most:
        t = t.clone(memory_format=torch.contiguous_format)
        return t, n, t.data_ptr()
    return t, s, p


def _scales_as_they_are(t: torch.Tensor, rows: int) -> bool:
    """Whether the kernels can read these scale bytes in place: 16 at a time, each of them in memory of the tensor's."""
    s, n = _row_stride(t), (t.shape[-1] + 15) // 16 * 16
    if s < t.shape[-1] or s % 16 or s > _STRIDE or t.data_ptr() % 16:
        return False
    return t.storage_offset() + max(rows - 1, 0) * s + n <= t.untyped_storage().nbytes()


def _sizes(rows: int, cols: int) -> None:
    if cols % 32 or not 32 <= cols <= _COLS:
        raise ValueError(f"{cols} columns: a multiple of 32 up to {_COLS}")
    if rows >= _ROWS:
        raise NotImplementedError(f"{rows} rows (below {_ROWS})")


class MXTensor:
    """Rows in microscaled blocks: `codes` uint8 (or float8_e4m3fn) [..., cols], for e2m1 [..., cols / 2] with the even
    value of a pair in the low four bits; `scales` uint8 (or float8_e8m0fnu) [..., cols / 32], E + 127 each; `fmt`
    "e4m3" or "e2m1".  Tensors whose rows the kernels can read where they are are kept, not copied."""

    __slots__ = ("_codes", "_scales", "_fmt", "_shape", "_device", "_buf", "_c", "_ref")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, fmt: str = "e4m3") -> None:
        bits = _bits(fmt)
        if codes.dtype != torch.uint8 and not (bits == 8 and codes.dtype == torch.float8_e4m3fn):
            raise ValueError(f"codes of dtype {codes.dtype} (uint8, for e4m3 also float8_e4m3fn)")
        if scales.dtype not in (torch.uint8, torch.float8_e8m0fnu):
            raise ValueError(f"scales of dtype {scales.dtype} (uint8 or float8_e8m0fnu)")
        if codes.device.type != "cuda" or scales.device != codes.device:
            raise ValueError("pgmoe blocks: codes and scales on one HIP device")
        if codes.dim() < 1 or codes.shape[-1] < 1:
            raise ValueError("codes: [..., cols]")
        cols, rows = codes.shape[-1] * 8 // bits, codes.numel() // codes.shape[-1]
        _sizes(rows, cols)
        if tuple(scales.shape) != (*codes.shape[:-1], cols // 32):
            raise ValueError(f"scales {tuple(scales.shape)} of codes {tuple(codes.shape)} ({fmt})")
        codes, stride, at = _placed(codes.view(torch.uint8), codes.shape[-1], 1, _STRIDE)
        scales = scales.view(torch.uint8)
        if not _scales_as_they_are(scales, rows):
            held = torch.empty(*scales.shape[:-1], (cols // 32 + 15) // 16 * 16, dtype=torch.uint8, device=scales.device)
            scales = held[..., :cols // 32].copy_(scales)
        self._codes, self._scales, self._buf = codes, scales, None
        self._set((*codes.shape[:-1], cols), fmt, codes.device,
                  Mx(at, scales.data_ptr(), stride, _row_stride(scales), rows, cols, bits))

    def _set(self, shape: Tuple[int, ...], fmt: str, device: torch.device, c: Mx) -> None:
        self._shape, self._fmt, self._device, self._c, self._ref = shape, fmt, device, c, ctypes.byref(c)

    @classmethod
    def _new(cls, shape: Tuple[int, ...], rows: int, fmt: str, device: torch.device) -> "MXTensor":
        """Blocks of a tensor of this shape, not yet written: one allocation, whose tensors are made when asked for."""
        bits, cols = _bits(fmt), shape[-1]
        _sizes(rows, cols)
        cs, ss = cols * bits >> 3, cols // 32 + 15 & -16
        t = cls.__new__(cls)
        t._codes = t._scales = None
        t._buf = torch.empty(rows * (cs + ss), dtype=torch.uint8, device=device)
        at = t._buf.data_ptr()
        t._set(shape, fmt, device, Mx(at, at + rows * cs, cs, ss, rows, cols, bits))
        return t

    def _rows_of(self, width: int, step: int, offset: int) -> torch.Tensor:
        if len(self._shape) == 2:
            return self._buf.as_strided((self._shape[0], width), (step, 1), offset)
        strides = [1]
        for n in reversed(self._shape[:-1]):
            strides.append(step)
            step *= n
        return self._buf.as_strided((*self._shape[:-1], width), strides[::-1], offset)

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._codes = self._rows_of(self._c.code_stride, self._c.code_stride, 0)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            c = self._c
            self._scales = self._rows_of(c.cols // 32, c.scale_stride, c.rows * c.code_stride)
        return self._scales

    # as they were given: the kernels read what the struct of them says
    fmt = property(lambda self: self._fmt)
    shape = property(lambda self: self._shape)
    device = property(lambda self: self._device)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values code * 2^E, each rounded once to `dtype` (fp32, fp16, bf16)."""
        if dtype not in _DT:
            raise NotImplementedError(f"values of dtype {dtype} (fp32, fp16 or bf16)")
        out = torch.empty(self._shape, dtype=dtype, device=self._device)
        if self._c.rows:
            launch(self._device, "pgmoe_mx_dequantize", lib().pgmoe_mx_dequantize, self._ref, out.data_ptr(), _DT[dtype])
        return out


def _floats(name: str, x: torch.Tensor) -> Tuple[torch.Tensor, int, int, int, int]:
    """(x or a copy that the kernels read, its type's code, its address, elements from row to row, rows)."""
    if not x.is_cuda:
        raise ValueError(f"{name}: a tensor on a HIP device")
    dt, shape = _DT.get(x.dtype), x.shape
    if dt is None:
        raise NotImplementedError(f"{name} of dtype {x.dtype} (fp32, fp16 or bf16)")
    if not shape or shape[-1] < 1:
        raise ValueError(f"{name}: [..., cols]")
    n = shape[-1]
    rows = x.numel() // n
    if rows >= _ROWS:
        raise NotImplementedError(f"{name}: {rows} rows (below {_ROWS})")
    x, stride, at = _placed(x, n, 4 if dt == 0 else 2, _FLOAT_STRIDE)
    return x, dt, at, stride, rows


def mx_quantize(x: torch.Tensor, fmt: str = "e4m3") -> MXTensor:
    """x [..., cols] (fp32, fp16, bf16) in blocks of 32 along its rows."""
    x, dt, at, stride, rows = _floats("x", x)
    dev = x.device
    y = MXTensor._new(tuple(x.shape), rows, fmt, dev)
    if rows:
        launch(dev, "pgmoe_mx_quantize", lib().pgmoe_mx_quantize, at, dt, stride, y._ref)
    return y


def exec_fused_act_mul_mx(gate: torch.Tensor, up: torch.Tensor, act: str = "silu", fmt: str = "e4m3") -> MXTensor:
    """act(gate) * up in blocks, act "silu" or "gelu" (tanh form), formed in fp32 from two tensors of one shape and type
    (the halves of a fused projection's output are taken as they are)."""
    code = _ACT.get(act)
    if code is None:
        raise NotImplementedError(f"activation {act!r} (silu or gelu)")
    if up.shape != gate.shape or up.dtype != gate.dtype or up.device != gate.device:
        raise ValueError(f"up {tuple(up.shape)} {up.dtype} beside gate {tuple(gate.shape)} {gate.dtype}: one shape, type and device")
    gate, dt, g, gs, rows = _floats("gate", gate)
    up, _, u, us, _ = _floats("up", up)
    dev = gate.device
    y = MXTensor._new(tuple(gate.shape), rows, fmt, dev)
    if rows:
        launch(dev, "pgmoe_mx_act_mul", lib().pgmoe_mx_act_mul, g, gs, u, us, dt, code, y._ref)
    return y


def _norm(x: torch.Tensor, delta: Optional[torch.Tensor], norm_weight: torch.Tensor, eps: float, fmt: str):
    x, dt, at, _, rows = _floats("x", x.contiguous())
    dev, shape = x.device, x.shape
    cols = shape[-1]
    d, ddt = None, 0
    if delta is not None:
        if delta.shape != shape or delta.device != dev:
            raise ValueError(f"delta {tuple(delta.shape)} on {delta.device} beside x {tuple(shape)} on {dev}")
        delta, ddt, d, _, _ = _floats("delta", delta.contiguous())
    w = norm_weight
    if w.numel() != cols:
        raise ValueError(f"norm weight has {w.numel()} elements, rows have {cols}")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    if w.dtype != torch.float32 or w.device != dev or not w.is_contiguous() or w.data_ptr() % 16:
        w = norm_weight.to(device=dev, dtype=torch.float32, copy=True).reshape(-1).contiguous()
    y = MXTensor._new(tuple(shape), rows, fmt, dev)
    h = torch.empty(shape, dtype=torch.float32, device=dev) if delta is not None else None
    if rows:
        launch(dev, "pgmoe_add_rmsnorm_mx", lib().pgmoe_add_rmsnorm_mx, at, dt, d, ddt, w.data_ptr(), eps,
               None if h is None else h.data_ptr(), y._ref)
    return h, y


def exec_fused_rmsnorm_mx(x: torch.Tensor, norm_weight: torch.Tensor, eps: float = 1e-6, fmt: str = "e4m3") -> MXTensor:
    """exec_fused_rmsnorm with its output in blocks; the values are formed in 64 bits and not rounded before."""
    return _norm(x, None, norm_weight, eps, fmt)[1]


def exec_fused_add_rmsnorm_mx(x: torch.Tensor, delta: torch.Tensor, norm_weight: torch.Tensor, eps: float = 1e-6,
                              fmt: str = "e4m3") -> Tuple[torch.Tensor, MXTensor]:
    """exec_fused_add_rmsnorm with its second output in blocks: (h = x.float() + delta.float(), RMSNorm(x + delta) * w), the
    second formed in 64 bits from the sum before its rounding to fp32."""
    return _norm(x, delta, norm_weight, eps, fmt)


def _gguf_blocks(raw: np.ndarray, rows: int, cols: int, device: torch.device) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of GGUF MXFP4 bytes: 17 a block, the scale's and 16 of codes, byte j holding values j (low) and
    j + 16 (high)."""
    b = torch.from_numpy(np.array(raw)).to(device).reshape(rows, cols // 32, 17)
    v = torch.cat((b[..., 1:] & 15, b[..., 1:] >> 4), -1)
    return (v[..., 0::2] | v[..., 1::2] << 4).reshape(rows, cols // 2), b[..., 0].contiguous()


class HipMXLinear(nn.Module):
    """y = x . W^T (+ bias) with W [out_features, in_features] in e2m1 blocks, laid out once for the matrix cores.

    forward(x, out_dtype=None): x an MXTensor [..., in_features] (either format), or fp32 / fp16 / bf16 values, which
    are brought to blocks of `act_fmt` first.  Products are summed in fp32 in a fixed order and rounded once, to
    out_dtype (fp32, fp16, bf16; by default x's, fp16 for an MXTensor).

    What a sum keeps: with e2m1 activations, fp32 outputs or up to 16 rows, products down to 2^-24 of their largest neighbour.
    16-bit outputs of more than 16 rows in e4m3 blocks are formed by the matrix cores' 8-bit products, which leave out what is
    below 2^-13 of the largest of 8 neighbouring ones (some 2e-5 of the outputs' 2-norm, a tenth of fp16's rounding): a row then
    differs by that from the same row in a call of up to 16.  fp32_sums=True takes the form of the few rows for all, at half
    the rate where rows are many."""

    def __init__(self, weight: MXTensor, bias: Optional[torch.Tensor] = None, act_fmt: str = "e4m3",
                 fp32_sums: bool = False) -> None:
        super().__init__()
        _bits(act_fmt)
        self._not_while_captured()
        if weight.fmt != "e2m1" or len(weight.shape) != 2 or weight.shape[0] < 1:
            raise ValueError(f"weight: e2m1 blocks [out_features, in_features], not {weight.fmt} {tuple(weight.shape)}")
        self.out_features, self.in_features = weight.shape
        self.device = weight.device
        self.act_fmt = act_fmt
        self.fp32_sums = bool(fp32_sums)
        if bias is not None and tuple(bias.shape) != (self.out_features,):
            raise ValueError(f"bias {tuple(bias.shape)} of {self.out_features} outputs")
        n = int(lib().pgmoe_mx_packed_bytes(self.out_features, self.in_features))
        if n < 0:
            raise NotImplementedError(f"weights of {self.out_features} x {self.in_features}")
        # no buffers of the module: its to() and half() would move or round what the kernel reads as given
        self._packed = torch.empty(n, dtype=torch.uint8, device=self.device)
        self._bias = None if bias is None else bias.detach().to(self.device, torch.float32, copy=True).contiguous()
        launch(self.device, "pgmoe_mx_pack", lib().pgmoe_mx_pack, weight._ref, self._packed.data_ptr())
        torch.cuda.current_stream(self.device).synchronize()  # from here on any stream may use them

    bias = property(lambda self: self._bias)

    @staticmethod
    def _not_while_captured() -> None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a layer is made before a graph is captured: its weights are laid out once, and waited for")

    @classmethod
    def from_gguf(cls, gguf_file: Any, weight_name: Union[str, Sequence[str]], bias_name: Optional[str] = None,
                  device: Union[torch.device, str] = "cuda", act_fmt: str = "e4m3", fp32_sums: bool = False) -> "HipMXLinear":
        """The named matrix; several names are one layer whose outputs follow each other.  MXFP4 tensors are kept
        exactly, F32 / F16 / BF16 ones are brought to e2m1 blocks."""
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("HipMXLinear runs on a HIP device (torch.device('cuda', i))")
        cls._not_while_captured()
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        codes, scales = [], []
        with _load_lock, torch.cuda.device(device):
            for name in [weight_name] if isinstance(weight_name, str) else weight_name:
                info = gguf_file.tensors[name]
                if len(info.shape) != 2:
                    raise ValueError(f"{name}: a matrix, not {tuple(info.shape)}")
                rows, cols, qt = int(info.shape[0]), int(info.shape[1]), int(info.qtype)
                if cols % 32:
                    raise ValueError(f"{name}: {cols} input features (a multiple of 32)")
                if qt == MXFP4:
                    c, s = _gguf_blocks(np.asarray(gguf_file.get_tensor_bytes(name)), rows, cols, device)
                elif qt in (F32, F16, BF16):
                    w = load_float_tensor(gguf_file, name, torch.device("cpu")).reshape(rows, cols)
                    t = mx_quantize(w.to(device, torch.float32), "e2m1")
                    c, s = t.codes, t.scales
                else:
                    raise NotImplementedError(f"{name}: ggml type {qt} (MXFP4, F32, F16 or BF16; GGUFQuantLinear takes the others)")
                codes.append(c)
                scales.append(s)
            bias = None
            if bias_name and bias_name in gguf_file.tensors:
                bias = load_float_tensor(gguf_file, bias_name, torch.device("cpu"))
            if len({c.shape[1] for c in codes}) != 1:
                raise ValueError("matrices of one layer have the same number of input features")
            return cls(MXTensor(torch.cat(codes), torch.cat(scales), "e2m1"), bias=bias, act_fmt=act_fmt, fp32_sums=fp32_sums)

    def forward(self, x: Union[torch.Tensor, MXTensor], out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        shape, n = x.shape, self.in_features
        if not shape or shape[-1] != n:
            raise ValueError(f"input of shape {tuple(shape)}, the layer has {n} input features")
        dev = self.device
        if x.device != dev:
            raise ValueError(f"input on {x.device}, the layer is on {dev}")
        given = isinstance(x, MXTensor)
        odt = out_dtype if out_dtype is not None else torch.float16 if given else x.dtype
        code = _DT.get(odt)
        if code is None:
            raise NotImplementedError(f"outputs of dtype {odt} (fp32, fp16 or bf16)")
        if self.fp32_sums:
            code += MX_FP32_SUMS
        if not given:
            x, dt, at, stride, rows = _floats("x", x)
        else:
            rows = x._c.rows
        out = torch.empty((*shape[:-1], self.out_features), dtype=odt, device=dev)
        if not rows:
            return out
        bias = None if self._bias is None else self._bias.data_ptr()
        if given:
            launch(dev, "pgmoe_mx_linear", lib().pgmoe_mx_linear, self._packed.data_ptr(), self.out_features, x._ref, bias,
                   out.data_ptr(), code)
            return out
        bits = _FMT[self.act_fmt]
        L = lib()
        nbytes = L.pgmoe_mx_linear_values_workspace_bytes(rows, n, bits)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None  # of this call alone
        launch(dev, "pgmoe_mx_linear_values", L.pgmoe_mx_linear_values, self._packed.data_ptr(), self.out_features,
               at, dt, stride, rows, n, bits, bias, out.data_ptr(), code,
               None if ws is None else ws.data_ptr(), nbytes)
        return out
