"""The global norm of many gradients, and clipping by it, on MI355X (``include/hsn_clip.h``):

    ``norm = sqrt(sum of g^2)`` over every element of every tensor, in float64,
    ``coefficient = min(1, max_norm / (norm + 1e-6))``, and 1 where the norm is infinite or NaN,
    ``out = coefficient g``.

:func:`norm` takes the norm, :func:`clip` scales too, in place or into other tensors, in two launches
for a list of up to 201 tensors. The gradients are fp32, bf16 or fp16, each of its own type, dense in
memory in any order of their dimensions. A norm that is not finite leaves the gradients as they are, so
that a program that sees it can skip its step. The coefficient is what
:func:`hsn_amd.trainer.scale64` takes. Every function requires ROCm tensors and the built HIP library;
there is no CPU path here. Nothing is kept between calls.
"""

from __future__ import annotations

import ctypes
import math
from collections.abc import Sequence
from typing import Optional

import torch
from torch import Tensor

from . import _lib
from ._lib import addr, call, call_on, called, native_calls, stream_of

__all__ = ["norm", "clip", "available"]

_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16,
          torch.bfloat16: _lib.DTYPE_BF16}


def _dense(t: Tensor) -> bool:
    """Whether the elements fill one run of memory, each once, in any order of the dimensions."""
    expected = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1),
                               key=lambda d: d[1]):
        if stride != expected and t.numel():
            return False
        expected *= size
    return True


def _one(t: Tensor, name: str, device) -> None:
    if not isinstance(t, Tensor):
        raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.device != device or t.dtype not in _DTYPE:
        raise ValueError(f"{name} must be float32, float16 or bfloat16 on {device}, got {t.dtype} on "
                         f"{t.device}")
    if t.layout != torch.strided or not _dense(t):
        raise ValueError(f"{name} must be dense in memory")
    if torch.is_grad_enabled() and t.requires_grad:
        raise ValueError(f"{name} requires a gradient, and there is none: call it under "
                         "torch.no_grad()")


def _run(grads: Sequence[Tensor], out: Optional[Sequence[Tensor]], max_norm: float):
    grads = grads if isinstance(grads, (list, tuple)) else list(grads)
    if out is not None and not isinstance(out, (list, tuple)):
        out = list(out)
    native = native_calls("hsn_clip_workspace", "hsn_clip")
    if native is not None and grads and isinstance(grads[0], Tensor) and grads[0].is_cuda:
        calls, size_at, call_at = native
        got = called(calls.grad_clip(size_at, call_at, stream_of(grads[0].device), grads, out, max_norm),
                     "hsn_clip")
        if got is not None:
            return got
    if not grads:
        raise ValueError("the list of gradients is empty")
    if not isinstance(grads[0], Tensor) or not grads[0].is_cuda:
        raise ValueError("the gradients must be ROCm device tensors")
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be 0 or more, got {max_norm}")
    dev, n = grads[0].device, len(grads)
    for i, g in enumerate(grads):
        _one(g, f"gradient {i}", dev)
    if out is not None:
        if len(out) != n:
            raise ValueError(f"out must have {n} tensors, got {len(out)}")
        for i, (o, g) in enumerate(zip(out, grads)):
            _one(o, f"out {i}", dev)
            strides = [(a, b) for size, a, b in zip(g.shape, g.stride(), o.stride()) if size > 1]
            if (o.dtype != g.dtype or o.shape != g.shape
                    or g.numel() and any(a != b for a, b in strides)):
                raise ValueError(f"out {i} must be laid out as its gradient, {tuple(g.shape)} "
                                 f"{g.dtype} with strides {g.stride()}, got {tuple(o.shape)} {o.dtype} "
                                 f"with strides {o.stride()}")
    pointers = ctypes.c_void_p * n
    numels = (ctypes.c_int64 * n)(*[g.numel() for g in grads])
    codes = (ctypes.c_int * n)(*[_DTYPE[g.dtype] for g in grads])
    ws_bytes = ctypes.c_int64(0)
    call("hsn_clip_workspace", numels, n, ctypes.byref(ws_bytes))
    result = torch.empty(2, dtype=torch.float64, device=dev)
    ws = torch.empty(ws_bytes.value, dtype=torch.uint8, device=dev)
    call_on(dev, "hsn_clip", pointers(*[addr(g) for g in grads]),
            None if out is None else pointers(*[addr(o) for o in out]), numels, codes, n,
            float(max_norm), result.data_ptr(), ws.data_ptr(), ws_bytes.value, stream_of(dev))
    for o in out or ():
        if not o.is_inference():
            torch.autograd.graph.increment_version(o)
    return result[0:1], result[1:2]


def norm(grads: Sequence[Tensor]) -> Tensor:
    """The norm of all the gradients together, ``[1]`` (float64, on their device)."""
    return _run(grads, None, math.inf)[0]


def clip(grads: Sequence[Tensor], max_norm: float, *,
         out: Optional[Sequence[Tensor]] = None) -> tuple[Tensor, Tensor]:
    """``(norm, coefficient)``, each ``[1]`` (float64): scales the gradients in place, which autograd
    counts as such, or into ``out``, whose tensors have the gradients' shapes, types and strides (some
    may be the gradients themselves). The product is taken in float64 and rounded to fp32, and from
    there to a 16-bit gradient's type. No tensor that is written may overlap another tensor of the
    call. In place, a coefficient of 1 leaves the memory untouched."""
    grads = grads if isinstance(grads, (list, tuple)) else list(grads)
    return _run(grads, grads if out is None else out, max_norm)


def available() -> bool:
    return _lib.available()
