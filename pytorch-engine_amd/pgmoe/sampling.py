"""The next token of each row of logits (pgmoe_sample): temperature, top-k, top-p, min-p.

    tokens, logprobs = sample_tokens(logits, u, temperature=0.8, top_k=40, top_p=0.95, min_p=0.05)

The step after the output head.  Random numbers are an input (u, one uniform number a row), so a run
repeats bit for bit: weights are summed in 64-bit fixed point, in which no order of sums shows.
Nothing synchronises with the host.  There is no CPU path.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple, Union

import torch

from ._lib import Sampling, lib
from .attention import launch

_DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_MAX_VOCAB = 1 << 20
_MAX_ROWS = 1 << 22


def _param(name: str, v: Union[float, int, torch.Tensor], rows: int, dev: torch.device, dtype: torch.dtype):
    """(kept tensor or None, scalar) of a sampling parameter: a number, or one value a row."""
    if isinstance(v, torch.Tensor):
        if v.device != dev or v.dtype != dtype or tuple(v.shape) != (rows,):
            raise ValueError(f"{name}: a number, or a {dtype} tensor [{rows}] on {dev}")
        return (v if v.stride(0) == 1 or rows == 1 else v.contiguous()), 0
    if not math.isfinite(v) or (dtype == torch.float32 and v < 0):
        raise ValueError(f"{name} must be finite and not negative")
    return None, v


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature: Union[float, torch.Tensor] = 1.0,
                  top_k: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
                  min_p: Union[float, torch.Tensor] = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(token int64 [rows], its log-probability fp32 [rows]) for logits [rows, vocab] (fp32, fp16, bf16).

    With w_i = exp((x_i - max x) / temperature) and the tokens ordered by logit (equal ones by index),
    the kept tokens are the shortest of: the first top_k (0: off); those before which the sum of w is
    below top_p times the whole (1: off); those with w >= min_p (0: off); one at least.  The whole is the
    row's, also where top_k is on: samplers that apply top_k first and take top_p of what is left keep fewer
    tokens at the same settings.  The token is the first in index order at which the sum of the kept w
    exceeds u times their total, u in [0, 1).  temperature 0: the largest logit.  Parameters: numbers, or a
    tensor of one value a row (float32; top_k int32).  w is held in multiples of 2^-s, s = min(51, 62 -
    ceil(log2(vocab))): a token with less than half of that is not drawn, not even at u = 0.  NaN and -inf
    logits are never drawn; a row that holds nothing else gives -1 and -inf."""
    if logits.device.type != "cuda" or logits.dim() != 2:
        raise ValueError("logits: [rows, vocab] on a HIP device")
    if logits.dtype not in _DT:
        raise NotImplementedError(f"logits of dtype {logits.dtype} (fp32, fp16 or bf16)")
    rows, vocab = logits.shape
    if not 1 <= vocab <= _MAX_VOCAB:
        raise NotImplementedError(f"vocabulary of {vocab} (1 .. {_MAX_VOCAB})")
    if rows > _MAX_ROWS:
        raise NotImplementedError(f"{rows} rows in one call (up to {_MAX_ROWS})")
    dev = logits.device
    if u.device != dev or u.dtype != torch.float32 or tuple(u.shape) != (rows,):
        raise ValueError(f"u: float32 [{rows}] on {dev}")
    if logits.stride(1) != 1 or (rows > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    if rows > 1 and u.stride(0) != 1:
        u = u.contiguous()
    t, tv = _param("temperature", temperature, rows, dev, torch.float32)
    k, kv = _param("top_k", top_k, rows, dev, torch.int32)
    p, pv = _param("top_p", top_p, rows, dev, torch.float32)
    m, mv = _param("min_p", min_p, rows, dev, torch.float32)
    par = Sampling(None if t is None else t.data_ptr(), None if k is None else k.data_ptr(),
                   None if p is None else p.data_ptr(), None if m is None else m.data_ptr(), tv, pv, mv,
                   0 if kv < 0 else min(int(kv), 2 ** 31 - 1))
    token = torch.empty(rows, dtype=torch.int64, device=dev)
    logprob = torch.empty(rows, dtype=torch.float32, device=dev)
    L = lib()
    n = int(L.pgmoe_sample_workspace_bytes(rows, vocab))
    ws = torch.empty(n, dtype=torch.uint8, device=dev)  # of this call alone
    launch(dev, "pgmoe_sample", L.pgmoe_sample, logits.data_ptr(), _DT[logits.dtype], logits.stride(0), rows, vocab,
           u.data_ptr(), ctypes.byref(par), token.data_ptr(), logprob.data_ptr(), ws.data_ptr(), n)
    return token, logprob
