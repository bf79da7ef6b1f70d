"""The choice of units in training on MI355X (``include/hsn_unit_router.h``): what
:func:`hsn_amd.unit_layer.unit_layer` chooses when it answers, with the gradient, and the balance loss
that keeps the units' loads alike. For each token the ``k`` largest of ``M`` logits and the softmax of
those; over all tokens, with ``c`` the times that a unit is chosen and ``p`` the softmax of all logits,

    ``balance = M sum_e (c_e / sum c) mean_i(p_ie)``,

1 where all units are chosen alike, differentiable through ``p``.

:func:`forward` and :func:`backward` are the two passes, :func:`choose_units` the same as one autograd
node. The logits are fp32, bf16 or fp16 ``[n, M]``, tokens any distance apart, ``M <= 256``, ``k <= 16``. A
unit whose logit is ``-inf`` is not chosen; a token without another, or with ``valid`` false, chooses
nothing, is not counted and has no gradient. Every function requires ROCm tensors and the built HIP
library; there is no CPU path here. Nothing is kept between calls.
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

__all__ = ["MAX_UNITS", "MAX_CHOSEN", "forward", "backward", "choose_units", "ChooseUnits", "available"]

MAX_UNITS, MAX_CHOSEN = 256, 16
_MAX_TOKENS = 1 << 30

_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16,
          torch.bfloat16: _lib.DTYPE_BF16}


def _logits(logits: Tensor, k: int, valid: Optional[Tensor]) -> tuple:
    """The checks of the inputs: ``(n, M, the tokens' distance, valid's address)``."""
    if not logits.is_cuda:
        raise ValueError(f"logits are on {logits.device}: the kernels take ROCm device tensors")
    if logits.dim() != 2 or logits.dtype not in _DTYPE:
        raise ValueError("logits must be [n, M] in float32, float16 or bfloat16, got "
                         f"{tuple(logits.shape)} {logits.dtype}")
    n, M = logits.shape
    if not 1 <= M <= MAX_UNITS or n >= _MAX_TOKENS:
        raise ValueError(f"M must be in [1, {MAX_UNITS}] and n below 2^30, got {M} and {n}")
    if not 1 <= k <= min(M, MAX_CHOSEN):
        raise ValueError(f"k must be in [1, {min(M, MAX_CHOSEN)}], got {k}")
    row, last = logits.stride()
    if last != 1 and M > 1:
        raise ValueError("a token's logits must be contiguous")
    return n, M, row, _dense(valid, "valid", (n,), torch.bool, logits.device)


def _dense(t: Optional[Tensor], name: str, shape: tuple, dtype: torch.dtype, device) -> Optional[int]:
    """The address of a contiguous tensor of this shape and type (``None`` for an absent one)."""
    if t is None:
        return None
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {shape} {dtype} on {device}, got {tuple(t.shape)} {t.dtype} "
                         f"on {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


@lru_cache(maxsize=1024)
def _workspace_bytes(n: int, M: int, dtype: int) -> int:
    out = ctypes.c_int64(0)
    call("hsn_unit_router_workspace", n, M, dtype, ctypes.byref(out))
    return out.value


def forward(logits: Tensor, k: int, *, valid: Optional[Tensor] = None) -> dict:
    """``units`` (int64) and ``shares`` (fp32) ``[n, k]`` of ``logits [n, M]``, the largest first and
    equal ones by unit, -1 and 0 in an empty slot; ``counts [M]`` (int64), ``probs [M]``, the
    probabilities' mean, and ``balance []`` (fp32); ``tally [M + 1]``, the counts and then the live
    tokens, for :func:`backward`. ``valid [n]`` is bool (``None``: all). A NaN logit is chosen first; a
    token with a NaN or ``+inf`` has NaN shares, and so are ``probs`` and ``balance`` then."""
    native = native_calls("hsn_unit_router_workspace", "hsn_unit_router_forward")
    if native is not None and logits.is_cuda:
        calls, size_at, call_at = native
        out = called(calls.unit_router_forward(size_at, call_at, stream_of(logits.device), logits, k,
                                               valid), "hsn_unit_router_forward")
        if out is not None:
            return dict(zip(("units", "shares", "balance", "counts", "probs", "tally"), out))
    n, M, row, valid_at = _logits(logits, k, valid)
    dev, code = logits.device, _DTYPE[logits.dtype]
    units = torch.empty((n, k), dtype=torch.int64, device=dev)
    shares = torch.empty((n, k), dtype=torch.float32, device=dev)
    tally = torch.empty(M + 1, dtype=torch.int64, device=dev)
    probs = torch.empty(M, dtype=torch.float32, device=dev)
    balance = torch.empty((), dtype=torch.float32, device=dev)
    size = _workspace_bytes(n, M, code)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    call_on(dev, "hsn_unit_router_forward", addr(logits), row, code, valid_at, units.data_ptr(),
            shares.data_ptr(), tally.data_ptr(), probs.data_ptr(), balance.data_ptr(), n, M, k,
            ws.data_ptr(), size, stream_of(dev))
    return {"units": units, "shares": shares, "balance": balance, "counts": tally[:M], "probs": probs,
            "tally": tally}


def backward(logits: Tensor, units: Tensor, tally: Tensor, d_shares: Optional[Tensor],
             d_balance: Optional[Tensor] = None, *, valid: Optional[Tensor] = None) -> Tensor:
    """``d_logits [n, M]``, contiguous and in the logits' type, from :func:`forward`'s inputs,
    ``units`` and ``tally``, and the cotangents ``d_shares [n, k]`` (fp32, a token's ``k`` contiguous)
    and ``d_balance`` (fp32, one element), either ``None`` where absent."""
    native = native_calls("hsn_unit_router_backward")
    if native is not None and logits.is_cuda:
        calls, call_at = native
        out = called(calls.unit_router_backward(call_at, stream_of(logits.device), logits, units, tally,
                                                d_shares, d_balance, valid), "hsn_unit_router_backward")
        if out is not None:
            return out
    if units.dim() != 2:
        raise ValueError(f"units must be [n, k], got {tuple(units.shape)}")
    k = units.shape[1]
    n, M, row, valid_at = _logits(logits, k, valid)
    dev = logits.device
    units_at = _dense(units, "units", (n, k), torch.int64, dev)
    tally_at = _dense(tally, "tally", (M + 1,), torch.int64, dev)
    g_row = 0
    if d_shares is not None:
        if (d_shares.shape != (n, k) or d_shares.dtype != torch.float32 or d_shares.device != dev
                or (d_shares.stride(1) != 1 and k > 1)):
            raise ValueError(f"d_shares must be {(n, k)} float32 on {dev}, a token's contiguous, got "
                             f"{tuple(d_shares.shape)} {d_shares.dtype} on {d_shares.device}")
        g_row = d_shares.stride(0)
    if d_balance is not None and (d_balance.numel() != 1 or d_balance.dtype != torch.float32
                                  or d_balance.device != dev):
        raise ValueError(f"d_balance must be one float32 on {dev}, got {tuple(d_balance.shape)} "
                         f"{d_balance.dtype} on {d_balance.device}")
    d_logits = torch.empty((n, M), dtype=logits.dtype, device=dev)
    call_on(dev, "hsn_unit_router_backward", addr(logits), row, _DTYPE[logits.dtype], valid_at,
            units_at, tally_at, addr(d_shares), g_row, addr(d_balance), d_logits.data_ptr(), n, M, k,
            stream_of(dev))
    return d_logits


class ChooseUnits(torch.autograd.Function):
    """:func:`forward` and :func:`backward` as one autograd node: ``apply(logits, k, valid)`` returns
    ``(shares, balance, units, tally)``, the first two with a gradient."""

    @staticmethod
    def forward(ctx, logits, k, valid):
        out = forward(logits, k, valid=valid)
        ctx.save_for_backward(logits, out["units"], out["tally"], valid)
        ctx.mark_non_differentiable(out["units"], out["tally"])
        ctx.set_materialize_grads(False)
        return out["shares"], out["balance"], out["units"], out["tally"]

    @staticmethod
    @once_differentiable
    def backward(ctx, d_shares, d_balance, *_):
        if d_shares is None and d_balance is None:
            return None, None, None
        logits, units, tally, valid = ctx.saved_tensors
        d_shares, d_balance = (None if d is None else d.resolve_neg() for d in (d_shares, d_balance))
        if d_shares is not None and d_shares.stride(1) != 1 and d_shares.shape[1] > 1:
            d_shares = d_shares.contiguous()  # an expanded cotangent (a sum's) has stride 0
        return backward(logits, units, tally, d_shares, d_balance, valid=valid), None, None


def choose_units(logits: Tensor, k: int, *,
                 valid: Optional[Tensor] = None) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """``(units [n, k], shares [n, k], balance [], counts [M])``; the shares and the balance are
    differentiable in ``logits``."""
    shares, balance, units, tally = ChooseUnits.apply(logits, k, valid)
    return units, shares, balance, tally[:-1]


def available() -> bool:
    return _lib.available()
