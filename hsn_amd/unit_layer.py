"""A whole layer of routed units for a few tokens on MI355X (``include/hsn_units_layer.h``): the
router's products, the choice of ``k`` units a token, the units and their weighted sum, without a
gradient. It is the answering side of the unit bank: the weights have the bank's ``[M, in, out]``
layout, and what bounds it is one read of the chosen units' weights.

:func:`unit_layer` requires ROCm tensors and the built HIP library; there is no CPU path here.
Nothing is kept between calls. For many tokens, or a gradient, there is the grouped unit MLP of
:mod:`hsn_amd.kernels.ops`.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional

import torch
from torch import Tensor

from . import _lib
from ._lib import addr, call, call_on, called, native_calls, stream_of

__all__ = ["MAX_TOKENS", "MAX_UNITS", "MAX_CHOSEN", "MAX_WIDTH", "unit_layer", "available"]

MAX_TOKENS, MAX_UNITS, MAX_CHOSEN = 64, 256, 16
MAX_WIDTH = 65536
ACTIVATIONS = {"gelu": 0, "swiglu": 1}
_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16,
          torch.bfloat16: _lib.DTYPE_BF16}


def _weight(t: Optional[Tensor], name: str, shape: tuple, dtype: torch.dtype, device) -> None:
    if t is None:
        return
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {shape} {dtype} on {device}, got {tuple(t.shape)} "
                         f"{t.dtype} on {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


@lru_cache(maxsize=1024)
def _workspace_bytes(n, M, k, d_in, H, d_out, dtype, activation) -> int:
    out = ctypes.c_int64(0)
    call("hsn_units_layer_workspace", n, M, k, d_in, H, d_out, dtype, activation, ctypes.byref(out))
    return out.value


def unit_layer(x: Tensor, router: Tensor, W1: Tensor, b1: Optional[Tensor], W2: Tensor,
               b2: Optional[Tensor], k: int, *, activation: str = "gelu") -> Tensor:
    """``y [n, d_out]``: for each token of ``x [n, d_in]`` (``n <= 64``) the ``k`` units with the
    largest products ``router x`` (``router [M, d_in]``, ``M <= 256``, ``k <= 16``; ties go to the
    lowest unit), the softmax ``p`` of those products, and ``sum_e p_e (v_e W2[e] + b2[e])`` with
    ``z = x W1[e] + b1[e]`` and ``v = gelu(z)`` (``W1 [M, d_in, H]``) or, for ``"swiglu"``,
    ``silu(z[:H]) z[H:]`` (``W1 [M, d_in, 2 H]``); ``W2 [M, H, d_out]``, biases optional. Everything
    has ``x``'s dtype (fp32, bf16 or fp16) and is computed in fp32; nothing is rounded before
    ``y``. ``x``'s rows may lie any distance apart."""
    native = native_calls("hsn_units_layer_workspace", "hsn_units_layer")
    if native is not None and x.is_cuda:
        calls, size_at, call_at = native
        out = called(calls.unit_layer(size_at, call_at, stream_of(x.device), x, router, W1, b1, W2, b2,
                                      k, ACTIVATIONS.get(activation, -1), int(activation == "swiglu")),
                     "hsn_units_layer")
        if out is not None:
            return out
    if not x.is_cuda:
        raise ValueError(f"x is on {x.device}: the kernels take ROCm device tensors")
    if x.dim() != 2 or x.dtype not in _DTYPE:
        raise ValueError("x must be [n, d_in] in float32, float16 or bfloat16, got "
                         f"{tuple(x.shape)} {x.dtype}")
    row, last = x.stride()
    if last != 1 and x.shape[1] > 1:
        raise ValueError("a row of x must be contiguous")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if W2.dim() != 3 or router.dim() != 2:
        raise ValueError("router must be [M, d_in] and W2 [M, H, d_out], got "
                         f"{tuple(router.shape)} and {tuple(W2.shape)}")
    n, d_in = x.shape
    M, H, d_out = W2.shape
    H1 = 2 * H if activation == "swiglu" else H
    if not 1 <= k <= min(M, MAX_CHOSEN):
        raise ValueError(f"k must be in [1, {min(M, MAX_CHOSEN)}], got {k}")
    if n > MAX_TOKENS or M > MAX_UNITS:
        raise ValueError(f"at most {MAX_TOKENS} tokens and {MAX_UNITS} units, got {n} and {M}")
    if max(d_in, H, d_out) > MAX_WIDTH:
        raise ValueError(f"widths of at most {MAX_WIDTH}, got d_in {d_in}, H {H} and d_out {d_out}")
    io, dev = x.dtype, x.device
    _weight(router, "router", (M, d_in), io, dev)
    _weight(W1, "W1", (M, d_in, H1), io, dev)
    _weight(b1, "b1", (M, H1), io, dev)
    _weight(W2, "W2", (M, H, d_out), io, dev)
    _weight(b2, "b2", (M, d_out), io, dev)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (x, router, W1, b1, W2, b2)):
        raise ValueError("unit_layer has no gradient: call it under torch.no_grad()")
    code, act = _DTYPE[io], ACTIVATIONS[activation]
    y = torch.empty((n, d_out), dtype=io, device=dev)
    size = _workspace_bytes(n, M, k, d_in, H, d_out, code, act)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    call_on(dev, "hsn_units_layer", addr(x), row, addr(router), addr(W1), addr(b1),
         addr(W2), addr(b2), y.data_ptr(), n, M, k, d_in, H, d_out, code, act, ws.data_ptr(),
         size, stream_of(dev))
    return y


def available() -> bool:
    return _lib.available()
