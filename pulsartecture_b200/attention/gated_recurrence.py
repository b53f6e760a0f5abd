"""Gated recurrent token mixer, the vector-state counterpart of TMLinKernelAttn.

    [x_t, g_t] = W u_t + b,  a_t = sigmoid(g_t)
    h_t = a_t h_{t-1} + (1 - a_t) x_t

Same contract as ``TMLinKernelAttn`` where they overlap: forward maps
(B, T, embed_dim) to (B, T, width) with an optional recurrent state in and
out, ``init_state`` and one-token ``step``. The projection is one library GEMM;
the recurrence runs in libfakla and reads both halves of its output in place.
The reference has no counterpart.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from ..backend.recurrence import gated_scan, gated_scan_step
from ..components.projections import LinearProjection


class GatedRecurrence(nn.Module):
    """h_t = a_t h_{t-1} + (1 - a_t) x_t over ``width`` channels (embed_dim by
    default). ``gate_bias`` is added to the gates' initial biases: 2 starts with
    memories of about eight tokens."""

    def __init__(self, embed_dim: int, width: Optional[int] = None, proj_bias: bool = True,
                 proj_init: str = "kaiming_uniform", gate_bias: float = 2.0, device=None, dtype=None):
        super().__init__()
        self.embed_dim = embed_dim
        self.width = width if width is not None else embed_dim
        if self.width < 1:
            raise ValueError(f"width must be at least 1, got {self.width}")
        self.proj = LinearProjection(embed_dim, 2 * self.width, use_bias=proj_bias, initialize=proj_init,
                                     device=device, dtype=dtype)
        if proj_bias:
            with torch.no_grad():
                self.proj.linear.bias[self.width:] += gate_bias

    def forward(self, x: torch.Tensor, state: Optional[torch.Tensor] = None, return_state: bool = False):
        """x (B, T, embed_dim) -> (B, T, width); with return_state also the state (B, width)."""
        value, gate = self.proj(x).chunk(2, dim=-1)
        out, final = gated_scan(value, gate, state, return_state=return_state)
        return (out, final) if return_state else out

    def init_state(self, batch: int, device=None) -> torch.Tensor:
        dev = device if device is not None else self.proj.linear.weight.device
        return torch.zeros(batch, self.width, device=dev, dtype=torch.float32)

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
        """One decode token per sequence: x (N, embed_dim) -> (N, width); state updated in place."""
        value, gate = self.proj(x).chunk(2, dim=-1)
        out, _ = gated_scan_step(value, gate, state)
        return out

    def extra_repr(self) -> str:
        return f"embed_dim={self.embed_dim}, width={self.width}"
