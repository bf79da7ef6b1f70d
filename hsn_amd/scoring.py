"""Log probabilities of given tokens on MI355X (``include/hsn_score.h``), with the entropy and the most
probable alternatives, and their gradient. For a row of logits ``l`` and its token ``t``, with ``log p =
l - max l - log(sum of exp(l - max l))``:

    ``logprob = log p[t]``,  ``entropy = -sum of p log p``.

:func:`forward` and :func:`backward` are the two passes, :func:`token_logprobs` the same as one
autograd node: a language model's loss is ``-logprob.mean()``. The logits are fp32, bf16 or fp16 with
rows any distance apart, and are read once each way; the passes make no ``[n, V]`` tensor but the
gradient. A token outside the vocabulary is skipped: its log probability is 0 and it has no gradient. A logit of
``-inf`` has no mass; a row of nothing else has the log probability ``-inf``, entropy 0 and no gradient. A
row with a NaN or ``+inf`` has NaN for its values and its gradient. Every function requires ROCm tensors
and the built HIP library; there is no CPU path here. Nothing is kept between calls.
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

__all__ = ["MAX_TOP", "MAX_TOKENS", "forward", "backward", "token_logprobs", "TokenLogprobs",
           "available"]

#: the most alternatives, and the largest vocabulary
MAX_TOP, MAX_TOKENS = 32, 1 << 24
_MAX_ROWS, _MAX_LOGITS = 1 << 24, 1 << 40

_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16,
          torch.bfloat16: _lib.DTYPE_BF16}
_TOKEN_BYTES = {torch.int64: 8, torch.int32: 4}


def _rows(logits: Tensor, tokens: Tensor) -> tuple:
    """The checks of the two inputs: ``(n, V, the rows' distance, the tokens' distance)``."""
    if not logits.is_cuda:
        raise ValueError(f"logits are on {logits.device}: the kernels take ROCm device tensors")
    if logits.dim() != 2 or logits.dtype not in _DTYPE:
        raise ValueError("logits must be [n, V] in float32, float16 or bfloat16, got "
                         f"{tuple(logits.shape)} {logits.dtype}")
    n, V = logits.shape
    if not 1 <= V <= MAX_TOKENS:
        raise ValueError(f"V must be in [1, {MAX_TOKENS}], got {V}")
    if n >= _MAX_ROWS or n * V >= _MAX_LOGITS:
        raise ValueError(f"fewer than 2^24 rows and 2^40 logits, got {n} rows of {V}")
    row, last = logits.stride()
    if last != 1 and V > 1:
        raise ValueError("a row of logits must be contiguous")
    if tokens.shape != (n,) or tokens.dtype not in _TOKEN_BYTES or tokens.device != logits.device:
        raise ValueError(f"tokens must be ({n},) int64 or int32 on {logits.device}, got "
                         f"{tuple(tokens.shape)} {tokens.dtype} on {tokens.device}")
    return n, V, row, tokens.stride(0)


@lru_cache(maxsize=1024)
def _workspace_bytes(n: int, V: int, dtype: int, top: int) -> int:
    out = ctypes.c_int64(0)
    call("hsn_score_workspace", n, V, dtype, top, ctypes.byref(out))
    return out.value


def forward(logits: Tensor, tokens: Tensor, *, top: int = 0, save: bool = True) -> dict:
    """``logprob`` and ``entropy`` ``[n]`` (fp32) of ``logits [n, V]`` and ``tokens [n]`` (int64 or
    int32); with ``top``, up to 32, also ``top_tokens`` (int64) and ``top_logprobs`` (fp32) ``[n, top]``,
    the largest logits first, equal ones by token, -1 and ``-inf`` where no further logit is above
    ``-inf`` (NaN is none of them); with ``save``, ``stats [n, 4]``, what :func:`backward` starts
    from. What is absent is ``None``."""
    native = native_calls("hsn_score_workspace", "hsn_score_forward")
    if native is not None and logits.is_cuda:
        calls, size_at, call_at = native
        out = called(calls.score_forward(size_at, call_at, stream_of(logits.device), logits, tokens,
                                         top, int(save)), "hsn_score_forward")
        if out is not None:
            return dict(zip(("logprob", "entropy", "top_tokens", "top_logprobs", "stats"), out))
    n, V, row, token_stride = _rows(logits, tokens)
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must be in [0, {MAX_TOP}], got {top}")
    dev, code = logits.device, _DTYPE[logits.dtype]

    def new(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device=dev)

    out = {"logprob": new(n), "entropy": new(n),
           "top_tokens": new(n, top, dtype=torch.int64) if top else None,
           "top_logprobs": new(n, top) if top else None, "stats": new(n, 4) if save else None}
    size = _workspace_bytes(n, V, code, top)
    ws = new(size, dtype=torch.uint8) if size else None
    call_on(dev, "hsn_score_forward", addr(logits), row, code, tokens.data_ptr(), token_stride,
            _TOKEN_BYTES[tokens.dtype], out["logprob"].data_ptr(), out["entropy"].data_ptr(),
            addr(out["top_tokens"]), addr(out["top_logprobs"]), addr(out["stats"]), n, V, top,
            addr(ws), size, stream_of(dev))
    return out


def _cotangent(t: Optional[Tensor], name: str, n: int, device) -> tuple:
    if t is None:
        return None, 0
    if t.shape != (n,) or t.dtype != torch.float32 or t.device != device:
        raise ValueError(f"{name} must be ({n},) float32 on {device}, got {tuple(t.shape)} {t.dtype} "
                         f"on {t.device}")
    return addr(t), t.stride(0)


def backward(logits: Tensor, tokens: Tensor, stats: Tensor, d_logprob: Optional[Tensor],
             d_entropy: Optional[Tensor] = None) -> Tensor:
    """``d_logits [n, V]``, contiguous and in the logits' type, from :func:`forward`'s inputs and
    ``stats`` and the cotangents ``[n]`` (fp32), either ``None`` where absent."""
    native = native_calls("hsn_score_backward")
    if native is not None and logits.is_cuda:
        calls, call_at = native
        out = called(calls.score_backward(call_at, stream_of(logits.device), logits, tokens, stats,
                                          d_logprob, d_entropy), "hsn_score_backward")
        if out is not None:
            return out
    n, V, row, token_stride = _rows(logits, tokens)
    dev = logits.device
    if (stats.shape != (n, 4) or stats.dtype != torch.float32 or stats.device != dev
            or not stats.is_contiguous()):
        raise ValueError(f"stats must be ({n}, 4) float32 on {dev}, contiguous, got "
                         f"{tuple(stats.shape)} {stats.dtype} on {stats.device}")
    g, g_stride = _cotangent(d_logprob, "d_logprob", n, dev)
    h, h_stride = _cotangent(d_entropy, "d_entropy", n, dev)
    d_logits = torch.empty((n, V), dtype=logits.dtype, device=dev)
    call_on(dev, "hsn_score_backward", addr(logits), row, _DTYPE[logits.dtype],
            tokens.data_ptr(), token_stride, _TOKEN_BYTES[tokens.dtype], addr(stats), g, g_stride,
            h, h_stride, d_logits.data_ptr(), n, V, stream_of(dev))
    return d_logits


class TokenLogprobs(torch.autograd.Function):
    """:func:`forward` and :func:`backward` as one autograd node: ``apply(logits, tokens)`` returns
    ``(logprob, entropy)``. The node keeps the logits and four numbers a row."""

    @staticmethod
    def forward(ctx, logits, tokens):
        out = forward(logits, tokens, save=ctx.needs_input_grad[0])
        ctx.save_for_backward(logits, tokens, out["stats"])
        ctx.set_materialize_grads(False)
        return out["logprob"], out["entropy"]

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logprob, d_entropy):
        if d_logprob is None and d_entropy is None:
            return None, None
        logits, tokens, stats = ctx.saved_tensors
        d_logprob, d_entropy = (None if d is None else d.resolve_neg() for d in (d_logprob, d_entropy))
        return backward(logits, tokens, stats, d_logprob, d_entropy), None


def token_logprobs(logits: Tensor, tokens: Tensor) -> tuple[Tensor, Tensor]:
    """``(logprob, entropy)`` of ``logits [..., V]`` and ``tokens [...]``, fp32 and of the tokens'
    shape, differentiable in ``logits``.

    Leading dimensions that are not rows of one distance are copied, and so is their gradient: the
    next-token slice ``logits[:, :-1]`` of several sequences is, where ``logits`` themselves with the
    tokens moved up and -1 behind the last are not."""
    if logits.dim() == 0 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens must be {tuple(logits.shape[:-1])}, got {tuple(tokens.shape)}")
    logprob, entropy = TokenLogprobs.apply(logits.reshape(tokens.numel(), logits.shape[-1]),
                                           tokens.reshape(-1))
    return logprob.view(tokens.shape), entropy.view(tokens.shape)


def available() -> bool:
    return _lib.available()
