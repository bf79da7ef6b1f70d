"""The gated linear recurrence over whole sequences on MI355X (``include/hsn_scan.h``): the
window's update ``h' = h + b (c - h)`` where every channel is written at every position,

    ``b = sigmoid(gate[r, t])``, ``c = tanh(y[r, t])`` or ``y[r, t]``,
    ``h[t] = (1 - b) (h[t-1], or 0 where reset[r, t]) + b c``,

with its backward, the carried state and its gradient, and the single position on a pool of states.
:func:`forward` and :func:`backward` are the two passes, :func:`gated_scan` the same as one
autograd node, :func:`step` one position of every running sequence.

``y`` and ``gate`` are ``[B, T, D]`` in fp32, bf16 or fp16; their last dimension is contiguous and
the other two may have any stride (slices of one fused product, a transposed batch). States and
their cotangents are fp32. Every function requires ROCm tensors and the built HIP library; there is
no CPU path here. Nothing is kept between calls.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor

from . import _lib
from ._lib import call, ptr, stream_of

__all__ = ["SPAN", "forward", "backward", "gated_scan", "GatedScan", "step", "available"]

#: positions between two of the states that :func:`forward` keeps for :func:`backward`
SPAN = 128

CANDIDATES = {"tanh": 0, "linear": 1}
_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16,
          torch.bfloat16: _lib.DTYPE_BF16}


def _candidate(name: str) -> int:
    if name not in CANDIDATES:
        raise ValueError(f"candidate must be one of {sorted(CANDIDATES)}, got {name!r}")
    return CANDIDATES[name]


def _dtype(t: Tensor, name: str) -> int:
    if t.dtype not in _DTYPE:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    return _DTYPE[t.dtype]


def _strided(t: Tensor, name: str, like: Tensor) -> None:
    """A tensor of the inputs' shape, type and device whose last dimension is contiguous."""
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be {tuple(like.shape)} {like.dtype} on {like.device}, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")


def _dense(t: Optional[Tensor], name: str, shape: tuple, dtype: torch.dtype, like: Tensor) -> None:
    if t is None:
        return
    if tuple(t.shape) != shape or t.dtype != dtype or t.device != like.device:
        raise ValueError(f"{name} must be {shape} {dtype} on {like.device}, got {tuple(t.shape)} "
                         f"{t.dtype} on {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _shape(y: Tensor, dims: int) -> tuple:
    if not y.is_cuda:
        raise ValueError(f"y is on {y.device}: the kernels take ROCm device tensors")
    if y.dim() != dims or y.shape[-1] == 0:
        raise ValueError(f"y must have {dims} dimensions and at least one channel, got "
                         f"{tuple(y.shape)}")
    return tuple(y.shape)


def _workspace(B: int, T: int, D: int, dtype: int, backward: int, device):
    out = ctypes.c_int64(0)
    call("hsn_scan_workspace", B, T, D, dtype, backward, ctypes.byref(out))
    n = out.value
    return (torch.empty(n, dtype=torch.uint8, device=device) if n else None), n


def forward(y: Tensor, gate: Tensor, reset: Optional[Tensor] = None, h0: Optional[Tensor] = None,
            *, candidate: str = "tanh", save: bool = True) -> dict:
    """The recurrence over a window: ``h [B, T, D]`` in ``y``'s dtype, the end state ``h_T [B, D]``
    (fp32) and, with ``save``, ``marks``: the states :func:`backward` starts from. ``reset [B, T]``
    is bool, ``h0 [B, D]`` fp32 (``None``: no resets, zero)."""
    B, T, D = _shape(y, 3)
    code, dev = _dtype(y, "y"), y.device
    _strided(y, "y", y)
    _strided(gate, "gate", y)
    _dense(reset, "reset", (B, T), torch.bool, y)
    _dense(h0, "h0", (B, D), torch.float32, y)
    h = torch.empty(B, T, D, dtype=y.dtype, device=dev)
    h_T = torch.empty(B, D, dtype=torch.float32, device=dev)
    marks = None
    if save:
        marks = torch.empty(B, -(-T // SPAN), D, dtype=torch.float32, device=dev)
    ws, ws_bytes = _workspace(B, T, D, code, 0, dev)
    call("hsn_scan_forward", ptr(y), y.stride(0), y.stride(1), ptr(gate), gate.stride(0),
         gate.stride(1), code, _candidate(candidate), ptr(reset), ptr(h0), ptr(h), ptr(h_T),
         ptr(marks), B, T, D, ptr(ws), ws_bytes, stream_of(dev))
    return {"h": h, "h_T": h_T, "marks": marks}


def backward(y: Tensor, gate: Tensor, marks: Tensor, reset: Optional[Tensor],
             d_h: Optional[Tensor], d_h_T: Optional[Tensor] = None, *,
             candidate: str = "tanh") -> tuple:
    """``(d_y, d_gate, d_h0)`` from :func:`forward`'s inputs and ``marks`` and the cotangents
    ``d_h [B, T, D]`` (``y``'s dtype) and ``d_h_T [B, D]`` (fp32), either ``None`` where absent.
    The cotangent of the state is fp32; ``d_y`` and ``d_gate`` have ``y``'s dtype."""
    B, T, D = _shape(y, 3)
    code, dev = _dtype(y, "y"), y.device
    _strided(y, "y", y)
    _strided(gate, "gate", y)
    _dense(marks, "marks", (B, -(-T // SPAN), D), torch.float32, y)
    _dense(reset, "reset", (B, T), torch.bool, y)
    _dense(d_h_T, "d_h_T", (B, D), torch.float32, y)
    row = pos = 0
    if d_h is not None:
        _strided(d_h, "d_h", y)
        row, pos = d_h.stride(0), d_h.stride(1)
    d_y = torch.empty(B, T, D, dtype=y.dtype, device=dev)
    d_gate = torch.empty_like(d_y)
    d_h0 = torch.empty(B, D, dtype=torch.float32, device=dev)
    ws, ws_bytes = _workspace(B, T, D, code, 1, dev)
    call("hsn_scan_backward", ptr(y), y.stride(0), y.stride(1), ptr(gate), gate.stride(0),
         gate.stride(1), code, _candidate(candidate), ptr(reset), ptr(marks), ptr(d_h), row, pos,
         ptr(d_h_T), ptr(d_y), ptr(d_gate), ptr(d_h0), B, T, D, ptr(ws), ws_bytes, stream_of(dev))
    return d_y, d_gate, d_h0


class GatedScan(torch.autograd.Function):
    """:func:`forward` and :func:`backward` as one autograd node with the carried state:
    ``apply(y, gate, h0, reset, candidate)`` returns ``(h, h_T)``. The node keeps ``y``, ``gate``
    and one fp32 state in :data:`SPAN` positions, not ``h``."""

    @staticmethod
    def forward(ctx, y, gate, h0, reset, candidate):
        out = forward(y, gate, reset, h0, candidate=candidate,
                      save=any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(y, gate, reset, out["marks"])
        ctx.candidate = candidate
        ctx.set_materialize_grads(False)
        return out["h"], out["h_T"]

    @staticmethod
    def backward(ctx, d_h, d_h_T):
        y, gate, reset, marks = ctx.saved_tensors
        if d_h is None and d_h_T is None:
            return None, None, None, None, None
        if d_h is not None and d_h.stride(-1) != 1 and d_h.shape[-1] > 1:
            d_h = d_h.contiguous()  # an expanded cotangent (a sum's) has stride 0
        if d_h_T is not None:
            d_h_T = d_h_T.contiguous()
        d_y, d_gate, d_h0 = backward(y, gate, marks, reset, d_h, d_h_T, candidate=ctx.candidate)
        return d_y, d_gate, (d_h0 if ctx.needs_input_grad[2] else None), None, None


def gated_scan(y: Tensor, gate: Tensor, reset: Optional[Tensor] = None,
               h0: Optional[Tensor] = None, *, candidate: str = "tanh") -> tuple[Tensor, Tensor]:
    """``(h, h_T)``, differentiable in ``y``, ``gate`` and ``h0``. A later window's loss reaches
    this one through ``h_T``; detach it to cut the segment."""
    return GatedScan.apply(y, gate, h0, reset, candidate)


def step(y: Tensor, gate: Tensor, state: Tensor, *, rows: Optional[Tensor] = None,
         reset: Optional[Tensor] = None, candidate: str = "tanh") -> Tensor:
    """One position of ``n`` running sequences, without a gradient: ``y``, ``gate`` ``[n, D]``; the
    states are the rows ``rows [n]`` (int32, distinct; ``None``: the first ``n``) of ``state
    [S, D]`` (fp32), updated in place. Returns the new states ``h [n, D]`` in ``y``'s dtype. A row
    outside ``[0, S)`` is padding: its ``h`` is zero and no state is touched."""
    n, D = _shape(y, 2)
    code = _dtype(y, "y")
    _strided(y, "y", y)
    _strided(gate, "gate", y)
    if state.dim() != 2:
        raise ValueError(f"state must be [S, {D}], got {tuple(state.shape)}")
    S = int(state.shape[0])
    _dense(state, "state", (S, D), torch.float32, y)
    _dense(rows, "rows", (n,), torch.int32, y)
    _dense(reset, "reset", (n,), torch.bool, y)
    h = torch.empty(n, D, dtype=y.dtype, device=y.device)
    call("hsn_scan_step", ptr(y), y.stride(0), ptr(gate), gate.stride(0), code,
         _candidate(candidate), ptr(rows), ptr(reset), ptr(state), ptr(h), n, S, D,
         stream_of(y.device))
    return h


def available() -> bool:
    return _lib.available()
