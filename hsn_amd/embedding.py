"""The embedding of tokens on MI355X (``include/hsn_embed.h``) and its gradient:

    ``out[i] = scale table[t_i]``,  ``d_table[v] = scale (sum of d_out[i] where t_i = v)``.

:func:`forward` and :func:`backward` are the two passes, :func:`embed` the same as one autograd node. The
table and the rows are fp32, bf16 or fp16, each its own (an fp32 table may give bf16 rows and take their
cotangents); sums are fp32 and rounded once, in an order that is the same every time. A token outside the
table is padding: a row of zeros, without a gradient. Every function requires ROCm tensors and the built
HIP library; there is no CPU path here. Nothing is kept between calls.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import addr, call, call_on, called, native_calls, stream_of

__all__ = ["MAX_TOKENS", "MAX_WIDTH", "forward", "backward", "embed", "Embed", "available"]

#: the largest table
MAX_TOKENS, MAX_WIDTH = 1 << 24, 65536
_MAX_POSITIONS = 1 << 26

_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16,
          torch.bfloat16: _lib.DTYPE_BF16}
_TOKEN_BYTES = {torch.int64: 8, torch.int32: 4}


def _rows_of(t: Tensor, dims: int) -> tuple:
    """``(B, T, the distances of rows and positions)`` of the first ``dims`` dimensions (two at most)."""
    if dims == 0:
        return 1, 1, 0, 0
    if dims == 1:
        return 1, t.shape[0], 0, t.stride(0)
    return t.shape[0], t.shape[1], t.stride(0), t.stride(1)


def _tokens(tokens: Tensor, device) -> None:
    if tokens.dtype not in _TOKEN_BYTES or tokens.device != device:
        raise ValueError(f"tokens must be int64 or int32 on {device}, got {tokens.dtype} on "
                         f"{tokens.device}")
    if tokens.numel() >= _MAX_POSITIONS:
        raise ValueError(f"fewer than 2^26 tokens, got {tokens.numel()}")


def _sizes(V: int, D: int) -> None:
    if not 1 <= V <= MAX_TOKENS or not 1 <= D <= MAX_WIDTH:
        raise ValueError(f"V must be in [1, {MAX_TOKENS}] and D in [1, {MAX_WIDTH}], got {V} and {D}")


def _type(dtype: torch.dtype) -> int:
    if dtype not in _DTYPE:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    return _DTYPE[dtype]


@lru_cache(maxsize=1024)
def _workspace_bytes(B: int, T: int, V: int, D: int, dtype: int) -> int:
    out = ctypes.c_int64(0)
    call("hsn_embed_workspace", B, T, V, D, dtype, ctypes.byref(out))
    return out.value


def forward(tokens: Tensor, table: Tensor, *, scale: float = 1.0,
            dtype: Optional[torch.dtype] = None) -> Tensor:
    """``[..., D]`` in ``dtype`` (``None``: the table's): the rows of ``table [V, D]`` (rows any distance
    apart) that ``tokens [...]`` (int64 or int32, any strides) name, times ``scale``."""
    dtype = table.dtype if dtype is None else dtype
    if tokens.dim() > 2:
        return forward(tokens.reshape(-1), table, scale=scale,
                       dtype=dtype).view(*tokens.shape, table.shape[-1])
    native = native_calls("hsn_embed_forward")
    if native is not None and table.is_cuda:
        calls, call_at = native
        out = called(calls.embed_forward(call_at, stream_of(table.device), tokens, table, scale,
                                         _DTYPE.get(dtype, -1)), "hsn_embed_forward")
        if out is not None:
            return out
    if not table.is_cuda:
        raise ValueError(f"table is on {table.device}: the kernels take ROCm device tensors")
    if table.dim() != 2 or table.dtype not in _DTYPE:
        raise ValueError("table must be [V, D] in float32, float16 or bfloat16, got "
                         f"{tuple(table.shape)} {table.dtype}")
    V, D = table.shape
    _sizes(V, D)
    if table.stride(1) != 1 and D > 1:
        raise ValueError("a row of the table must be contiguous")
    dev = table.device
    _tokens(tokens, dev)
    code = _type(dtype)
    B, T, stride_b, stride_t = _rows_of(tokens, tokens.dim())
    out = torch.empty((*tokens.shape, D), dtype=dtype, device=dev)
    call_on(dev, "hsn_embed_forward", tokens.data_ptr(), stride_b, stride_t, _TOKEN_BYTES[tokens.dtype],
            addr(table), table.stride(0), _DTYPE[table.dtype], float(scale), out.data_ptr(), code, B,
            T, V, D, stream_of(dev))
    return out


def backward(tokens: Tensor, d_out: Tensor, V: int, *, scale: float = 1.0,
             dtype: Optional[torch.dtype] = None) -> Tensor:
    """``d_table [V, D]`` in ``dtype`` (``None``: the cotangents'), contiguous, from the tokens ``[...]``
    and ``d_out [..., D]`` (the last dimension contiguous, any other strides)."""
    dtype = d_out.dtype if dtype is None else dtype
    if tokens.dim() > 2 and d_out.shape[:-1] == tokens.shape:
        return backward(tokens.reshape(-1), d_out.reshape(tokens.numel(), d_out.shape[-1]), V, scale=scale,
                        dtype=dtype)
    native = native_calls("hsn_embed_workspace", "hsn_embed_backward")
    if native is not None and d_out.is_cuda:
        calls, size_at, call_at = native
        out = called(calls.embed_backward(size_at, call_at, stream_of(d_out.device), tokens, d_out, V,
                                          scale, _DTYPE.get(dtype, -1)), "hsn_embed_backward")
        if out is not None:
            return out
    if not d_out.is_cuda:
        raise ValueError(f"d_out is on {d_out.device}: the kernels take ROCm device tensors")
    if d_out.dtype not in _DTYPE or d_out.dim() == 0 or d_out.shape[:-1] != tokens.shape:
        raise ValueError(f"d_out must be {(*tokens.shape, 'D')} in float32, float16 or bfloat16, got "
                         f"{tuple(d_out.shape)} {d_out.dtype}")
    D = d_out.shape[-1]
    _sizes(V, D)
    if d_out.stride(-1) != 1 and D > 1:
        raise ValueError("d_out's last dimension must be contiguous")
    dev = d_out.device
    _tokens(tokens, dev)
    code = _type(dtype)
    B, T, stride_b, stride_t = _rows_of(tokens, tokens.dim())
    _, _, row_b, row_t = _rows_of(d_out, tokens.dim())
    size = _workspace_bytes(B, T, V, D, _DTYPE[d_out.dtype])
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    d_table = torch.empty((V, D), dtype=dtype, device=dev)
    call_on(dev, "hsn_embed_backward", tokens.data_ptr(), stride_b, stride_t, _TOKEN_BYTES[tokens.dtype],
            addr(d_out), row_b, row_t, _DTYPE[d_out.dtype], float(scale), d_table.data_ptr(), code, B,
            T, V, D, ws.data_ptr(), size, stream_of(dev))
    return d_table


class Embed(torch.autograd.Function):
    """:func:`forward` and :func:`backward` as one autograd node: ``apply(tokens, table, scale, dtype)``.
    The node keeps the tokens."""

    @staticmethod
    def forward(ctx, tokens, table, scale, dtype):
        ctx.save_for_backward(tokens)
        ctx.V, ctx.table_dtype, ctx.scale = table.shape[0], table.dtype, scale
        return forward(tokens, table, scale=scale, dtype=dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        tokens, = ctx.saved_tensors
        d_out = d_out.resolve_neg()
        if d_out.stride(-1) != 1 and d_out.shape[-1] > 1:
            d_out = d_out.contiguous()  # an expanded cotangent (a sum's) has stride 0
        return None, backward(tokens, d_out, ctx.V, scale=ctx.scale, dtype=ctx.table_dtype), None, None


def embed(tokens: Tensor, table: Tensor, *, scale: float = 1.0,
          dtype: Optional[torch.dtype] = None) -> Tensor:
    """:func:`forward`, differentiable in ``table``."""
    return Embed.apply(tokens, table, scale, dtype)


def available() -> bool:
    return _lib.available()
