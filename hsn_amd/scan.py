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
no CPU path here. Nothing is kept between calls. A call's checks, allocations and launch are one step
of the host helper ``hsn_amd._calls`` where it is built; without it, and for arguments it declines,
the same checks run here, where each mismatch has its message.
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


def _first(y: Tensor, dims: int) -> tuple:
    """The checks of ``y``: ``(its shape, dtype code, dtype, device)``, which the others must have."""
    if not y.is_cuda:
        raise ValueError(f"y is on {y.device}: the kernels take ROCm device tensors")
    shape, dtype = y.shape, y.dtype
    if len(shape) != dims or shape[-1] == 0:
        raise ValueError(f"y must have {dims} dimensions and at least one channel, got "
                         f"{tuple(shape)}")
    if dtype not in _DTYPE:
        raise ValueError(f"y must be float32, float16 or bfloat16, got {dtype}")
    if max(shape) >= _lib.SIZE_LIMIT:
        raise ValueError(f"sizes are below 2^31, got {tuple(shape)}")
    return shape, _DTYPE[dtype], dtype, y.device


def _strides(t: Tensor, name: str, shape, dtype, device) -> tuple:
    """The strides of a tensor of the inputs' shape, type and device whose last dimension is
    contiguous."""
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {tuple(shape)} {dtype} on {device}, got {tuple(t.shape)} "
                         f"{t.dtype} on {t.device}")
    strides = t.stride()
    if strides[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    return strides


def _dense(t: Optional[Tensor], name: str, shape: tuple, dtype: torch.dtype, device) -> Optional[int]:
    """The address of a contiguous tensor of this shape and type (``None`` for an absent one)."""
    if t is None:
        return None
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {tuple(shape)} {dtype} on {device}, got {tuple(t.shape)} "
                         f"{t.dtype} on {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


@lru_cache(maxsize=1024)
def _workspace_bytes(B: int, T: int, D: int, dtype: int, backward: int) -> int:
    out = ctypes.c_int64(0)
    call("hsn_scan_workspace", B, T, D, dtype, backward, ctypes.byref(out))
    return out.value


def _workspace(B: int, T: int, D: int, dtype: int, backward: int, device):
    n = _workspace_bytes(B, T, D, dtype, backward)
    return (torch.empty(n, dtype=torch.uint8, device=device) if n else None), n


def forward(y: Tensor, gate: Tensor, reset: Optional[Tensor] = None, h0: Optional[Tensor] = None,
            *, candidate: str = "tanh", save: bool = True) -> dict:
    """The recurrence over a window: ``h [B, T, D]`` in ``y``'s dtype, the end state ``h_T [B, D]``
    (fp32) and, with ``save``, ``marks``: the states :func:`backward` starts from. ``reset [B, T]``
    is bool, ``h0 [B, D]`` fp32 (``None``: no resets, zero)."""
    native = native_calls("hsn_scan_workspace", "hsn_scan_forward")
    if native is not None and y.is_cuda:
        calls, size_at, call_at = native
        out = called(calls.scan_forward(size_at, call_at, stream_of(y.device), y, gate, reset, h0,
                                        CANDIDATES.get(candidate, -1), int(save), SPAN),
                     "hsn_scan_forward")
        if out is not None:
            return {"h": out[0], "h_T": out[1], "marks": out[2]}
    shape, code, io, dev = _first(y, 3)
    B, T, D = shape
    ys, gs = _strides(y, "y", shape, io, dev), _strides(gate, "gate", shape, io, dev)
    reset_at = _dense(reset, "reset", (B, T), torch.bool, dev)
    h0_at = _dense(h0, "h0", (B, D), torch.float32, dev)
    h = torch.empty(shape, dtype=io, device=dev)
    h_T = torch.empty((B, D), dtype=torch.float32, device=dev)
    marks = None
    if save:
        marks = torch.empty((B, -(-T // SPAN), D), dtype=torch.float32, device=dev)
    ws, ws_bytes = _workspace(B, T, D, code, 0, dev)
    call_on(dev, "hsn_scan_forward", y.data_ptr(), ys[0], ys[1], gate.data_ptr(), gs[0], gs[1], code,
         _candidate(candidate), reset_at, h0_at, h.data_ptr(), h_T.data_ptr(), addr(marks), B, T, D,
         addr(ws), ws_bytes, stream_of(dev))
    return {"h": h, "h_T": h_T, "marks": marks}


def backward(y: Tensor, gate: Tensor, marks: Tensor, reset: Optional[Tensor],
             d_h: Optional[Tensor], d_h_T: Optional[Tensor] = None, *,
             candidate: str = "tanh") -> tuple:
    """``(d_y, d_gate, d_h0)`` from :func:`forward`'s inputs and ``marks`` and the cotangents
    ``d_h [B, T, D]`` (``y``'s dtype) and ``d_h_T [B, D]`` (fp32), either ``None`` where absent.
    The cotangent of the state is fp32; ``d_y`` and ``d_gate`` have ``y``'s dtype."""
    native = native_calls("hsn_scan_workspace", "hsn_scan_backward")
    if native is not None and y.is_cuda:
        calls, size_at, call_at = native
        out = called(calls.scan_backward(size_at, call_at, stream_of(y.device), y, gate, marks, reset,
                                         d_h, d_h_T, CANDIDATES.get(candidate, -1), SPAN),
                     "hsn_scan_backward")
        if out is not None:
            return out
    shape, code, io, dev = _first(y, 3)
    B, T, D = shape
    ys, gs = _strides(y, "y", shape, io, dev), _strides(gate, "gate", shape, io, dev)
    marks_at = _dense(marks, "marks", (B, -(-T // SPAN), D), torch.float32, dev)
    reset_at = _dense(reset, "reset", (B, T), torch.bool, dev)
    d_h_T_at = _dense(d_h_T, "d_h_T", (B, D), torch.float32, dev)
    ds = (0, 0) if d_h is None else _strides(d_h, "d_h", shape, io, dev)
    d_y = torch.empty(shape, dtype=io, device=dev)
    d_gate = torch.empty(shape, dtype=io, device=dev)
    d_h0 = torch.empty((B, D), dtype=torch.float32, device=dev)
    ws, ws_bytes = _workspace(B, T, D, code, 1, dev)
    call_on(dev, "hsn_scan_backward", y.data_ptr(), ys[0], ys[1], gate.data_ptr(), gs[0], gs[1], code,
         _candidate(candidate), reset_at, marks_at, addr(d_h), ds[0], ds[1], d_h_T_at,
         d_y.data_ptr(), d_gate.data_ptr(), d_h0.data_ptr(), B, T, D, addr(ws), ws_bytes,
         stream_of(dev))
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
    @once_differentiable
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
    [S, D]`` (fp32), updated in place, which autograd counts as such. Returns the new states ``h [n, D]``
    in ``y``'s dtype. A row outside ``[0, S)`` is padding: its ``h`` is zero and no state is touched."""
    native = native_calls("hsn_scan_step")
    if native is not None and y.is_cuda:
        calls, call_at = native
        out = called(calls.scan_step(call_at, stream_of(y.device), y, gate, state, rows, reset,
                                     CANDIDATES.get(candidate, -1)), "hsn_scan_step")
        if out is not None:
            return out
    shape, code, io, dev = _first(y, 2)
    n, D = shape
    ys, gs = _strides(y, "y", shape, io, dev), _strides(gate, "gate", shape, io, dev)
    S = state.shape[0] if state.dim() == 2 else -1
    if S >= _lib.SIZE_LIMIT:
        raise ValueError(f"sizes are below 2^31, got a pool of {S} states")
    state_at = _dense(state, "state", (S, D), torch.float32, dev)
    rows_at = _dense(rows, "rows", (n,), torch.int32, dev)
    reset_at = _dense(reset, "reset", (n,), torch.bool, dev)
    if torch.is_grad_enabled() and (y.requires_grad or gate.requires_grad or state.requires_grad):
        raise ValueError("step has no gradient: call it under torch.no_grad()")
    h = torch.empty(shape, dtype=io, device=dev)
    call_on(dev, "hsn_scan_step", y.data_ptr(), ys[0], gate.data_ptr(), gs[0], code, _candidate(candidate),
         rows_at, reset_at, state_at, h.data_ptr(), n, S, D, stream_of(dev))
    if n and not state.is_inference():
        torch.autograd.graph.increment_version(state)
    return h


def available() -> bool:
    return _lib.available()
