"""Gated linear recurrence on libfakla (torch-tensor front end).

    a_t = sigmoid(gate_t) or gate_t
    h_t = a_t h_{t-1} + (1 - a_t) x_t    or    a_t h_{t-1} + x_t

per batch row and channel: the elementwise counterpart of FA-KLA's recurrence
(a vector state instead of a matrix per head), with the same hand-off of an
fp32 state between calls. The reference has no counterpart.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .interface import _check_device, _dtype_code, _needs_grad, _ptr, _require, _stream

GATE_ACTIVATIONS = {"sigmoid": _lib.FAKLA_ACT_SIGMOID, "identity": _lib.FAKLA_ACT_IDENTITY}


def _check_gated(x: torch.Tensor, gate: torch.Tensor, state: Optional[torch.Tensor], gate_act: str, ndim: int):
    """Checks shared by the scan and the step: the device and the dtype code."""
    shape = "(B, T, D)" if ndim == 3 else "(N, D)"
    _require(x.dim() == ndim and gate.dim() == ndim, f"x and gate must be {shape}")
    _require(x.shape == gate.shape, f"x {tuple(x.shape)} and gate {tuple(gate.shape)} shapes must match")
    _require(x.dtype == gate.dtype, "x and gate must have the same dtype")
    _require(gate_act in GATE_ACTIVATIONS, f"unknown gate_act {gate_act!r}; choose from {sorted(GATE_ACTIVATIONS)}")
    dev = _check_device([x, gate, state], ["x", "gate", "state"])
    if state is not None:
        expected = (x.shape[0], x.shape[-1])
        _require(tuple(state.shape) == expected, f"state must be {expected}, got {tuple(state.shape)}")
        _require(state.dtype == torch.float32, "state must be float32")
    return dev, _dtype_code(x)


def _dense_channels(t: torch.Tensor) -> torch.Tensor:
    """t with unit stride over its channels (other strides are free)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


class _GatedScanFn(torch.autograd.Function):
    """fakla_gated_scan with gradients (fakla_gated_scan_backward)."""

    @staticmethod
    def forward(ctx, x, gate, state, act, mix):
        ctx.set_materialize_grads(False)
        out, final, saved = _run_scan(x, gate, state, act, mix, True, True)
        ctx.save_for_backward(x, gate, saved)
        ctx.act, ctx.mix, ctx.has_state = act, mix, state is not None
        return out, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dfinal):
        x, gate, saved = ctx.saved_tensors
        B, T, D = x.shape
        dev = x.device
        dout = torch.zeros(B, T, D, device=dev, dtype=x.dtype) if dout is None else dout.contiguous().to(dtype=x.dtype)
        dfinal = None if dfinal is None else dfinal.contiguous().float()
        dx = torch.empty(B, T, D, device=dev, dtype=x.dtype)
        dgate = torch.empty_like(dx)
        dstate = torch.empty(B, D, device=dev, dtype=torch.float32) if ctx.has_state else None
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().fakla_gated_scan_backward(
                _ptr(x), _ptr(gate), _ptr(saved), _ptr(dout), _ptr(dfinal), _ptr(dx), _ptr(dgate), _ptr(dstate),
                B, T, D, x.stride(0), x.stride(1), gate.stride(0), gate.stride(1), ctx.act, ctx.mix,
                _dtype_code(x), _stream(dev)))
        return dx, dgate, dstate, None, None


def _run_scan(x, gate, state, act, mix, return_state, save):
    B, T, D = x.shape
    dev = x.device
    out = torch.empty(B, T, D, device=dev, dtype=x.dtype)
    final = torch.empty(B, D, device=dev, dtype=torch.float32) if return_state else None
    L = _lib.lib()
    saved = None
    if save:
        saved = torch.empty(L.fakla_gated_scan_saved_bytes(B, T, D), device=dev, dtype=torch.uint8)
    with torch.cuda.device(dev):
        _lib.check(L.fakla_gated_scan(
            _ptr(x), _ptr(gate), _ptr(out), _ptr(state), _ptr(final), _ptr(saved), B, T, D,
            x.stride(0), x.stride(1), gate.stride(0), gate.stride(1), act, mix, _dtype_code(x), _stream(dev)))
    return out, final, saved


def gated_scan(x: torch.Tensor, gate: torch.Tensor, state: Optional[torch.Tensor] = None, *,
               gate_act: str = "sigmoid", mix: bool = True,
               return_state: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """h_t = a_t h_{t-1} + b_t over (B, T, D): returns ``(h, final state)`` (or ``(h, None)``).

    x, gate: (B, T, D), float32 or bfloat16; column blocks of a wider tensor
    (``proj.chunk(2, -1)``) and expanded batch or time dimensions are read in
    place. gate_act: "sigmoid" (a = sigmoid(gate)) or "identity" (a = gate, a
    decay factor: products of 128 consecutive ones have to fit float32).
    mix: b = (1 - a) x, otherwise b = x. state: (B, D) float32, h before the
    first token, or None for zero; it is not modified. h is carried in float32
    and rounded to the input dtype in the output; the final state (B, D) is
    float32. Differentiable in x, gate and state, through both results.

    A gate of -inf ("sigmoid") or 0 ("identity") forgets the state, so packed
    documents are separated by setting it at their first tokens.
    """
    dev, _ = _check_gated(x, gate, state, gate_act, 3)
    B, T, D = x.shape
    act, mix = GATE_ACTIVATIONS[gate_act], bool(mix)
    if B * T * D == 0:
        final = None
        if return_state:
            final = state.clone() if state is not None else torch.zeros(B, D, device=dev, dtype=torch.float32)
        return torch.empty(B, T, D, device=dev, dtype=x.dtype), final
    x, gate = _dense_channels(x), _dense_channels(gate)
    state = None if state is None else state.contiguous()
    if _needs_grad(x, gate, state):
        out, final = _GatedScanFn.apply(x, gate, state, act, mix)
        return out, (final if return_state else None)
    out, final, _ = _run_scan(x, gate, state, act, mix, return_state, False)
    return out, final


def gated_scan_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, *, gate_act: str = "sigmoid",
                    mix: bool = True, new_state: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token of ``gated_scan`` for N sequences; returns ``(h (N, D), state)``.

    x, gate: (N, D); state: (N, D) float32, contiguous. ``state`` is updated in
    place, or with ``new_state`` (float32, (N, D), contiguous, not overlapping
    it) left as it is and the new one written there. Not differentiable.
    """
    _require(state is not None, "state is required")
    dev, code = _check_gated(x, gate, state, gate_act, 2)
    _require(not _needs_grad(x, gate, state, new_state), "gated_scan_step has no backward; use gated_scan, or torch.no_grad()")
    target = state if new_state is None else new_state
    _require(target.device == dev and target.shape == state.shape and target.dtype == torch.float32,
             "new_state must be a float32 tensor like state, on the same device")
    _require(state.is_contiguous() and target.is_contiguous(), "state and new_state must be contiguous")
    N, D = x.shape
    out = torch.empty(N, D, device=dev, dtype=x.dtype)
    if N * D == 0:
        return out, target
    x, gate = _dense_channels(x), _dense_channels(gate)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().fakla_gated_scan_step(
            _ptr(x), _ptr(gate), _ptr(out), _ptr(state), _ptr(target), N, D, x.stride(0), gate.stride(0),
            GATE_ACTIVATIONS[gate_act], bool(mix), code, _stream(dev)))
    return out, target
