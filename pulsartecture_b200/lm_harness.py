"""End-to-end language-model harness around FA-KLA.

The reference ships no model: ultra_rwka/models/full.py, base_model.py,
variants/* and configs/* are empty files. This module is this package's own
composition of reference-style parts with FA-KLA (`TMLinKernelAttn`, default
elu+1 map) running on libfakla, and is labelled as such wherever it is
measured:

    x = embed(ids)
    L x [ x += W_o TMLinKernelAttn(LN(x));  x += MoE(LN(x)) ]
    logits = head(LN(x))

Layers named in ``recurrent_layers`` take GatedRecurrence in the place of
TMLinKernelAttn. ``score``, ``loss`` and ``distill_loss`` go on from the logits
with ``token_logprobs`` and ``distill_topk``.

The MoE layer follows the reference's top-k gating (ultra_rwka/MoE/gating.py:
112-145: the top-k gate logits, a softmax over those k, no noise at
inference) over GELU MLP experts (the shape of ultra_rwka/MoE/branches.py
MLPBranch). The reference's IDAM memory and wavelet mixing are left out: the
repository gives them no defaults, and the wavelet projection needs a
backend operation the reference does not implement.

Everything but the token mixing and what follows the logits runs on PyTorch /
cuBLAS; the attention sublayers are the FA-KLA kernels of this package, the
recurrent ones its gated scan.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch
import torch.nn as nn
import torch.nn.functional as F

from .attention import GatedRecurrence, TMLinKernelAttn
from .backend.logits import TokenLogprobs, distill_topk, token_logprobs
from .kernels import LearnablePositiveMap


class MoEFeedForward(nn.Module):
    """Top-k of n_experts GELU MLPs (d_model -> d_ff -> d_model), weights = a
    softmax over the k largest gate logits (gating.py:136-144)."""

    def __init__(self, d_model: int, d_ff: int, n_experts: int = 8, top_k: int = 2, device=None, dtype=None):
        super().__init__()
        if not 1 <= top_k <= n_experts:
            raise ValueError(f"top_k must be in [1, n_experts], got {top_k}")
        fk = {"device": device, "dtype": dtype}
        self.n_experts, self.top_k = n_experts, top_k
        self.gate = nn.Linear(d_model, n_experts, bias=False, **fk)
        self.w_in = nn.Parameter(torch.empty(n_experts, d_ff, d_model, **fk))
        self.b_in = nn.Parameter(torch.zeros(n_experts, d_ff, **fk))
        self.w_out = nn.Parameter(torch.empty(n_experts, d_model, d_ff, **fk))
        self.b_out = nn.Parameter(torch.zeros(n_experts, d_model, **fk))
        for e in range(n_experts):
            nn.init.kaiming_uniform_(self.w_in[e], a=math.sqrt(5))
            nn.init.kaiming_uniform_(self.w_out[e], a=math.sqrt(5))

    def routing(self, x2: torch.Tensor):
        """(rows, d) -> expert indices (rows, k) and weights (rows, k)."""
        logits = self.gate(x2)
        top_logits, top_idx = torch.topk(logits, self.top_k, dim=-1)
        weights = F.softmax(top_logits.float(), dim=-1).to(x2.dtype)
        return top_idx, weights

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        lead = x.shape[:-1]
        x2 = x.reshape(-1, x.shape[-1])
        idx, w = self.routing(x2)
        out = torch.zeros_like(x2)
        flat_idx = idx.reshape(-1)
        flat_w = w.reshape(-1)
        tok = torch.arange(x2.shape[0], device=x.device).repeat_interleave(self.top_k)
        order = torch.argsort(flat_idx)
        counts = torch.bincount(flat_idx, minlength=self.n_experts).tolist()
        start = 0
        for e, n in enumerate(counts):
            if n == 0:
                continue
            sel = order[start:start + n]
            start += n
            rows = tok[sel]
            h = F.gelu(F.linear(x2[rows], self.w_in[e], self.b_in[e]))
            y = F.linear(h, self.w_out[e], self.b_out[e])
            out.index_add_(0, rows, y * flat_w[sel, None])
        return out.reshape(*lead, -1)


class FaklaBlock(nn.Module):
    """Pre-norm block: FA-KLA attention or a gated recurrence (with an output
    projection back to d_model) and an MoE feed-forward, each added to the
    residual stream."""

    def __init__(self, d_model: int, n_heads: int, head_dim: int, d_ff: int, n_experts: int, top_k: int,
                 device=None, dtype=None, recurrent: bool = False):
        super().__init__()
        fk = {"device": device, "dtype": dtype}
        feat = n_heads * head_dim
        self.ln_attn = nn.LayerNorm(d_model, **fk)
        if recurrent:
            self.attn = GatedRecurrence(d_model, feat, **fk)
        else:
            self.attn = TMLinKernelAttn(d_model, LearnablePositiveMap(feat, feat, **fk), num_heads=n_heads,
                                        qk_dim=head_dim, v_dim=head_dim, **fk)
        self.proj_out = nn.Linear(feat, d_model, **fk)
        self.ln_ff = nn.LayerNorm(d_model, **fk)
        self.ff = MoEFeedForward(d_model, d_ff, n_experts, top_k, **fk)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x = x + self.proj_out(self.attn(self.ln_attn(x)))
        return x + self.ff(self.ln_ff(x))


class FaklaLM(nn.Module):
    """Token ids (B, T) -> next-token logits (B, T, vocab). Defaults: 12
    layers, d_model 1024, 16 FA-KLA heads of 64, top-2 of 8 experts with
    d_ff 4096, vocabulary 32000. ``recurrent_layers``: indices of the layers
    that mix tokens by a gated recurrence instead of FA-KLA."""

    def __init__(self, vocab: int = 32000, d_model: int = 1024, n_layers: int = 12, n_heads: int = 16,
                 head_dim: int = 64, d_ff: int = 4096, n_experts: int = 8, top_k: int = 2, device=None,
                 dtype=None, recurrent_layers: Sequence[int] = ()):
        super().__init__()
        fk = {"device": device, "dtype": dtype}
        recurrent = set(recurrent_layers)
        if not recurrent <= set(range(n_layers)):
            raise ValueError(f"recurrent_layers {sorted(recurrent)} are not all in [0, {n_layers})")
        self.embed = nn.Embedding(vocab, d_model, **fk)
        self.blocks = nn.ModuleList([FaklaBlock(d_model, n_heads, head_dim, d_ff, n_experts, top_k, **fk,
                                                recurrent=i in recurrent) for i in range(n_layers)])
        self.ln_f = nn.LayerNorm(d_model, **fk)
        self.head = nn.Linear(d_model, vocab, bias=False, **fk)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        x = self.embed(ids)
        for blk in self.blocks:
            x = blk(x)
        return self.head(self.ln_f(x))

    @torch.no_grad()
    def score(self, ids: torch.Tensor, top_k: int = 0, temperature: float = 1.0,
              ignore_index: int = -100) -> TokenLogprobs:
        """What the model gave the tokens ids[:, 1:] in their places: (B, T - 1)
        log probabilities and entropies, with the top_k alternatives of each.
        Padding (ids of ignore_index) is embedded as token 0 and has log
        probability 0; entropies and alternatives are given there too."""
        logits = self(ids.masked_fill(ids == ignore_index, 0))
        return token_logprobs(logits[:, :-1], ids[:, 1:], top_k=top_k, temperature=temperature,
                              ignore_index=ignore_index)

    def loss(self, ids: torch.Tensor, entropy_weight: float = 0.0, ignore_index: int = -100) -> torch.Tensor:
        """Mean next-token cross entropy of ids (B, T), less entropy_weight times
        the mean entropy over the same positions. Targets equal to ignore_index
        (padding) are left out; such ids are embedded as token 0."""
        targets = torch.cat([ids[:, 1:], torch.full_like(ids[:, :1], ignore_index)], dim=1)
        counted = targets != ignore_index
        r = token_logprobs(self(ids.masked_fill(ids == ignore_index, 0)), targets, ignore_index=ignore_index)
        total = r.logprobs.sum()
        if entropy_weight:
            total = total + entropy_weight * r.entropy.masked_fill(~counted, 0.0).sum()
        return -total / counted.sum().clamp_min(1)

    def distill_loss(self, ids: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                     teacher_lse: Optional[torch.Tensor] = None, temperature: float = 1.0,
                     ignore_index: int = -100) -> torch.Tensor:
        """Mean KL divergence from a teacher's largest logits, teacher_ids and
        teacher_logits (B, T, K), over the positions of ids (B, T) that have an
        entry (an id that is not -1). Padding (ids of ignore_index) is embedded
        as token 0 and left out."""
        padding = ids == ignore_index
        teacher_ids = teacher_ids.masked_fill(padding[..., None], -1)
        losses = distill_topk(self(ids.masked_fill(padding, 0)), teacher_ids, teacher_logits, teacher_lse,
                              temperature=temperature)
        return losses.sum() / (teacher_ids != -1).any(-1).sum().clamp_min(1)
