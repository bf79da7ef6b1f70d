"""The choice of a token from logits on MI355X (``include/hsn_sample.h``): temperature, top-k, top-p
and min-p, from given random numbers.

:func:`sample` takes the settings as numbers for the whole batch or as tensors with one a row, so a
batch may hold requests of different kinds. The random numbers are the caller's: the same numbers
give the same tokens, on every run and in every batch (a token's weight is a fixed-point number, so
sums do not depend on their order). It requires ROCm tensors and the built HIP library; there is no
CPU path here. Nothing is kept between calls.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Union

import torch
from torch import Tensor

from . import _lib
from ._lib import addr, call, call_on, called, native_calls, stream_of

__all__ = ["MAX_TOKENS", "sample", "available"]

#: the largest vocabulary
MAX_TOKENS = 262144

_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16,
          torch.bfloat16: _lib.DTYPE_BF16}


class _Settings(ctypes.Structure):
    _fields_ = [("temperature", ctypes.c_float), ("top_k", ctypes.c_int32),
                ("top_p", ctypes.c_float), ("min_p", ctypes.c_float)]


def _setting(v, name: str, dtype: torch.dtype, n: int, device):
    """``(the address of a setting's row values, its value for all rows)``."""
    if not isinstance(v, Tensor):
        return None, v
    if v.shape != (n,) or v.dtype != dtype or v.device != device:
        raise ValueError(f"{name} must be a number or ({n},) {dtype} on {device}, got "
                         f"{tuple(v.shape)} {v.dtype} on {v.device}")
    if not v.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return addr(v), 0


@lru_cache(maxsize=1024)
def _workspace_bytes(n: int, V: int, dtype: int) -> int:
    out = ctypes.c_int64(0)
    call("hsn_sample_workspace", n, V, dtype, ctypes.byref(out))
    return out.value


def sample(logits: Tensor, u: Tensor, *, temperature: Union[float, Tensor] = 1.0,
           top_k: Union[int, Tensor] = 0, top_p: Union[float, Tensor] = 1.0,
           min_p: Union[float, Tensor] = 0.0) -> Tensor:
    """Tokens ``[n]`` (int64) from ``logits [n, V]`` (fp32, bf16 or fp16, rows any distance apart)
    and ``u [n]`` (fp32, in ``[0, 1)``).

    With the logits over ``temperature``: the ``top_k`` largest are kept (0: all; ties go to the
    lowest token), of these the shortest prefix, from the largest on, that holds ``top_p`` of their
    mass, and of these the ones with at least ``min_p`` of the largest's; the largest always is.
    The token is the first kept one, in the order of tokens, at which the running share of the kept
    mass exceeds ``u``. A temperature of 0 gives the largest logit's first token. NaN counts as
    ``-inf``; a row without a logit above ``-inf`` gives -1. The settings are numbers, or tensors of
    ``n`` (``top_k`` int32, the others fp32)."""
    native = native_calls("hsn_sample_workspace", "hsn_sample")
    if native is not None and logits.is_cuda:
        calls, size_at, call_at = native
        out = called(calls.sample(size_at, call_at, stream_of(logits.device), logits, u, temperature,
                                  top_k, top_p, min_p), "hsn_sample")
        if out is not None:
            return out
    if not logits.is_cuda:
        raise ValueError(f"logits are on {logits.device}: the kernels take ROCm device tensors")
    if logits.dim() != 2 or logits.dtype not in _DTYPE:
        raise ValueError("logits must be [n, V] in float32, float16 or bfloat16, got "
                         f"{tuple(logits.shape)} {logits.dtype}")
    n, V = logits.shape
    dev = logits.device
    if not 1 <= V <= MAX_TOKENS:
        raise ValueError(f"V must be in [1, {MAX_TOKENS}], got {V}")
    if n >= _lib.SIZE_LIMIT:
        raise ValueError(f"sizes are below 2^31, got {n} rows")
    row, last = logits.stride()
    if last != 1 and V > 1:
        raise ValueError("a row of logits must be contiguous")
    if u.shape != (n,) or u.dtype != torch.float32 or u.device != dev:
        raise ValueError(f"u must be ({n},) float32 on {dev}, got {tuple(u.shape)} {u.dtype} on "
                         f"{u.device}")
    if not u.is_contiguous():
        raise ValueError("u must be contiguous")
    t_at, t = _setting(temperature, "temperature", torch.float32, n, dev)
    k_at, k = _setting(top_k, "top_k", torch.int32, n, dev)
    p_at, p = _setting(top_p, "top_p", torch.float32, n, dev)
    m_at, m = _setting(min_p, "min_p", torch.float32, n, dev)
    if not 0 <= k < 2 ** 31:
        raise ValueError(f"top_k must be in [0, 2^31), got {k}")
    code = _DTYPE[logits.dtype]
    size = _workspace_bytes(n, V, code)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    tokens = torch.empty(n, dtype=torch.int64, device=dev)
    call_on(dev, "hsn_sample", addr(logits), row, code, addr(u), t_at, k_at, p_at, m_at,
         ctypes.byref(_Settings(t, k, p, m)), tokens.data_ptr(), n, V, addr(ws), size,
         stream_of(dev))
    return tokens


def available() -> bool:
    return _lib.available()
