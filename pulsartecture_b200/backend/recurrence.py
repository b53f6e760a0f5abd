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
from .interface import _launch, _ptr

GATE_ACTIVATIONS = {"sigmoid": _lib.FAKLA_ACT_SIGMOID, "identity": _lib.FAKLA_ACT_IDENTITY}
_DTYPES = {torch.float32: _lib.FAKLA_F32, torch.bfloat16: _lib.FAKLA_BF16}


def _check_gated(x: torch.Tensor, gate: torch.Tensor, state: Optional[torch.Tensor], gate_act: str, ndim: int):
    """Checks shared by the scan and the step; returns the device, the dtype
    code and the gate activation's."""
    if x.dim() != ndim or gate.dim() != ndim:
        raise RuntimeError(f"x and gate must be {'(B, T, D)' if ndim == 3 else '(N, D)'}")
    if x.shape != gate.shape:
        raise RuntimeError(f"x {tuple(x.shape)} and gate {tuple(gate.shape)} shapes must match")
    if x.dtype != gate.dtype:
        raise RuntimeError("x and gate must have the same dtype")
    act = GATE_ACTIVATIONS.get(gate_act)
    if act is None:
        raise RuntimeError(f"unknown gate_act {gate_act!r}; choose from {sorted(GATE_ACTIVATIONS)}")
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise RuntimeError(f"gated_scan supports float32 and bfloat16 inputs, got {x.dtype}")
    dev = x.device
    if dev.type != "cuda":
        raise RuntimeError("x must be a CUDA tensor (libfakla has no CPU path)")
    if gate.device != dev or (state is not None and state.device != dev):
        raise RuntimeError(f"x, gate and state must be on one device ({dev})")
    if state is not None:
        if state.dim() != 2 or state.shape[0] != x.shape[0] or state.shape[1] != x.shape[-1]:
            raise RuntimeError(f"state must be {(x.shape[0], x.shape[-1])}, got {tuple(state.shape)}")
        if state.dtype != torch.float32:
            raise RuntimeError("state must be float32")
    return dev, code, act


def _dense_channels(t: torch.Tensor) -> torch.Tensor:
    """t with unit stride over its channels (other strides are free)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


class _GatedScanFn(torch.autograd.Function):
    """fakla_gated_scan with gradients (fakla_gated_scan_backward)."""

    @staticmethod
    def forward(ctx, x, gate, state, act, mix, code):
        ctx.set_materialize_grads(False)
        out, final, saved = _run_scan(x, gate, state, act, mix, code, True, True)
        ctx.save_for_backward(x, gate, saved)
        ctx.form = act, mix, code, state is not None
        return out, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dfinal):
        x, gate, saved = ctx.saved_tensors
        act, mix, code, has_state = ctx.form
        B, T, D = x.shape
        dev = x.device
        dout = torch.zeros((B, T, D), device=dev, dtype=x.dtype) if dout is None else dout.contiguous()
        dx, dgate = torch.empty_like(dout), torch.empty_like(dout)
        dstate = torch.empty((B, D), device=dev, dtype=torch.float32) if has_state else None
        dfinal = None if dfinal is None else dfinal.contiguous()
        xb, xt, _ = x.stride()
        gb, gt, _ = gate.stride()
        _launch(dev, _lib.lib().fakla_gated_scan_backward, _ptr(x), _ptr(gate), _ptr(saved), _ptr(dout), _ptr(dfinal),
                _ptr(dx), _ptr(dgate), _ptr(dstate), B, T, D, xb, xt, gb, gt, act, mix, code)
        return dx, dgate, dstate, None, None, None


def _run_scan(x, gate, state, act, mix, code, return_state, save):
    B, T, D = x.shape
    dev = x.device
    L = _lib.lib()
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    final = torch.empty((B, D), device=dev, dtype=torch.float32) if return_state else None
    saved = torch.empty(L.fakla_gated_scan_saved_bytes(B, T, D), device=dev, dtype=torch.uint8) if save else None
    xb, xt, _ = x.stride()
    gb, gt, _ = gate.stride()
    _launch(dev, L.fakla_gated_scan, _ptr(x), _ptr(gate), _ptr(out), _ptr(state), _ptr(final), _ptr(saved), B, T, D,
            xb, xt, gb, gt, act, mix, code)
    return out, final, saved


def gated_scan(x: torch.Tensor, gate: torch.Tensor, state: Optional[torch.Tensor] = None, *,
               gate_act: str = "sigmoid", mix: bool = True,
               return_state: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """h_t = a_t h_{t-1} + b_t over (B, T, D): returns ``(h, final state)`` (or ``(h, None)``).

    x, gate: (B, T, D), float32 or bfloat16; column blocks of a wider tensor
    (``proj.chunk(2, -1)``) and expanded batch or time dimensions are read in
    place. gate_act: "sigmoid" (a = sigmoid(gate)) or "identity" (a = gate, a
    decay factor: products of up to 64 consecutive ones have to fit float32;
    bfloat16 has none between 1 - 2^-8 and 1, so slower decays need float32 x
    and gate). mix: b = (1 - a) x, otherwise b = x. state: (B, D) float32, h
    before the first token, or None for zero; it is not modified. h is carried
    in float32 and rounded to the input dtype in the output; the final state
    (B, D) is float32. Differentiable in x, gate and state, through both results.

    A gate of -inf ("sigmoid") or 0 ("identity") forgets the state, so packed
    documents are separated by setting it at their first tokens.
    """
    dev, code, act = _check_gated(x, gate, state, gate_act, 3)
    mix = bool(mix)
    if x.numel() == 0:
        B, _, D = x.shape
        final = None
        if return_state:
            final = state.clone() if state is not None else torch.zeros(B, D, device=dev, dtype=torch.float32)
        return x * gate, final  # nothing, but with x and gate behind it
    x, gate = _dense_channels(x), _dense_channels(gate)
    state = None if state is None else state.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or
                                    (state is not None and state.requires_grad)):
        out, final = _GatedScanFn.apply(x, gate, state, act, mix, code)
        return out, (final if return_state else None)
    out, final, _ = _run_scan(x, gate, state, act, mix, code, return_state, False)
    return out, final


def gated_scan_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, *, gate_act: str = "sigmoid",
                    mix: bool = True, new_state: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token of ``gated_scan`` for N sequences; returns ``(h (N, D), state)``.

    x, gate: (N, D); state: (N, D) float32, contiguous. ``state`` is updated in
    place, or with ``new_state`` (float32, (N, D), contiguous, not overlapping
    it) left as it is and the new one written there. Not differentiable.
    """
    if state is None:
        raise RuntimeError("state is required")
    dev, code, act = _check_gated(x, gate, state, gate_act, 2)
    target = state if new_state is None else new_state
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or state.requires_grad or target.requires_grad):
        raise RuntimeError("gated_scan_step has no backward; use gated_scan, or torch.no_grad()")
    if target is not state and (target.device != dev or target.shape != state.shape or target.dtype != torch.float32):
        raise RuntimeError("new_state must be a float32 tensor like state, on the same device")
    if not (state.is_contiguous() and target.is_contiguous()):
        raise RuntimeError("state and new_state must be contiguous")
    N, D = x.shape
    out = torch.empty((N, D), device=dev, dtype=x.dtype)
    if N * D == 0:
        return out, target
    x, gate = _dense_channels(x), _dense_channels(gate)
    _launch(dev, _lib.lib().fakla_gated_scan_step, _ptr(x), _ptr(gate), _ptr(out), _ptr(state), _ptr(target), N, D,
            x.stride(0), gate.stride(0), act, bool(mix), code)
    return out, target
