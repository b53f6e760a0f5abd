"""Scoring and distilling rows of logits on libfakla (torch-tensor front end).

``token_logprobs`` (log probabilities of given tokens, entropies, the most
probable tokens) and ``distill_topk`` (KL divergence from a teacher known by
its largest logits) each read the logits once, and once more in the backward;
no probabilities are stored. The reference has no counterpart.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .interface import _launch, _ptr

MAX_TOP_K = 32
MAX_ENTRIES = 256
_DTYPES = {torch.float32: _lib.FAKLA_F32, torch.bfloat16: _lib.FAKLA_BF16}


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor                 # (...) float32
    entropy: torch.Tensor                  # (...) float32
    top_logprobs: Optional[torch.Tensor]   # (..., top_k) float32, or None
    top_ids: Optional[torch.Tensor]        # (..., top_k) int64, or None


def _as_rows(logits: torch.Tensor):
    """logits, and how its rows lie: (batch, rows, vocab, batch stride, row
    stride). A view wherever the leading dimensions come down to two strides (a
    slice of positions or of a padded vocabulary does), a dense copy otherwise."""
    nd = logits.dim()
    if nd > 3:
        logits = logits.reshape(-1, *logits.shape[-2:])
        nd = 3
    st = logits.stride()
    if st[-1] != 1 and logits.shape[-1] != 1:
        logits = logits.contiguous()
        st = logits.stride()
    if nd == 3:
        return logits, (*logits.shape, st[0], st[1])
    if nd == 2:
        return logits, (1, *logits.shape, 0, st[0])
    return logits, (1, 1, *logits.shape, 0, 0)


def _check_rows(logits: torch.Tensor, temperature: float):
    """Returns the leading shape, the dtype code and the temperature."""
    temperature = float(temperature)
    if not 1e-30 <= temperature <= 1e30:
        raise RuntimeError(f"temperature must be positive (1e-30 to 1e30), got {temperature}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise RuntimeError("logits must be (..., vocab)")
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise RuntimeError(f"logits must be float32 or bfloat16, got {logits.dtype}")
    if not logits.is_cuda:
        raise RuntimeError("logits must be a CUDA tensor (libfakla has no CPU path)")
    return logits.shape[:-1], code, temperature


class _TokenLogprobsFn(torch.autograd.Function):
    """fakla_token_logprobs with gradients (fakla_token_logprobs_backward)."""

    @staticmethod
    def forward(ctx, logits, targets, top_k, temperature, ignore_index, code):
        ctx.set_materialize_grads(False)
        rows, at = _as_rows(logits)
        lp, ent, top, ids, stats = _run_logprobs(rows, at, targets, top_k, temperature, ignore_index, code, True)
        ctx.save_for_backward(rows, targets, stats, ent, ids)
        ctx.form = at, top_k, temperature, ignore_index, code, logits.shape
        if top_k:
            ctx.mark_non_differentiable(ids)
        return lp, ent, top, ids

    @staticmethod
    @once_differentiable
    def backward(ctx, dlp, dent, dtop, _):
        rows, targets, stats, ent, ids = ctx.saved_tensors
        at, top_k, temperature, ignore_index, code, shape = ctx.form
        dlp, dent, dtop = (None if t is None else t.contiguous() for t in (dlp, dent, dtop))
        dlogits = torch.empty_like(rows, memory_format=torch.contiguous_format).view(shape)
        _launch(rows.device, _lib.lib().fakla_token_logprobs_backward, _ptr(rows), _ptr(targets), _ptr(stats), _ptr(ent),
                _ptr(ids), _ptr(dlp), _ptr(dent), _ptr(dtop), _ptr(dlogits), *at, top_k, temperature, ignore_index, code)
        return dlogits, None, None, None, None, None


def _run_logprobs(rows, at, targets, top_k, temperature, ignore_index, code, save):
    dev, lead = rows.device, targets.shape
    lp = torch.empty_like(targets, dtype=torch.float32)
    ent = torch.empty_like(lp)
    top = torch.empty((*lead, top_k), device=dev, dtype=torch.float32) if top_k else None
    ids = torch.empty((*lead, top_k), device=dev, dtype=torch.int64) if top_k else None
    stats = torch.empty((at[0] * at[1], 2), device=dev, dtype=torch.float32) if save else None
    _launch(dev, _lib.lib().fakla_token_logprobs, _ptr(rows), _ptr(targets), _ptr(lp), _ptr(ent), _ptr(top), _ptr(ids),
            _ptr(stats), *at, top_k, temperature, ignore_index, code)
    return lp, ent, top, ids, stats


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, top_k: int = 0, temperature: float = 1.0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of ``targets`` under softmax(logits / temperature), the
    entropy of each row in nats, and its ``top_k`` most probable tokens.

    logits: (..., vocab), float32 or bfloat16, vocab up to 2^20; a slice of
    positions (``logits[:, :-1]``) or of a padded vocabulary is read in place.
    targets: (...) int64. Returns ``TokenLogprobs(logprobs, entropy,
    top_logprobs, top_ids)``, all float32 but the ids: descending, the lower
    index first among equals; None without top_k (at most 32).

    A target equal to ``ignore_index`` gives log probability 0 and no gradient
    through it; the row's entropy and alternatives are still given. Another
    target outside of the vocabulary gives NaN and is reported by
    ``device_status``. A row of nothing but -inf has log probabilities -inf,
    entropy 0 and a zero gradient; one with a NaN or +inf gives NaN and ids -1.

    Differentiable in logits through the three float results. To train on next
    tokens, put ignore_index at the last position's target rather than slicing
    the logits: a slice's gradient is copied once more by autograd.
    """
    lead, code, temperature = _check_rows(logits, temperature)
    if targets.shape != lead:
        raise RuntimeError(f"targets {tuple(targets.shape)} do not go with logits {tuple(logits.shape)}")
    if targets.dtype != torch.int64:
        raise RuntimeError("targets must be int64")
    if targets.device != logits.device:
        raise RuntimeError(f"targets are on {targets.device}, expected {logits.device}")
    if not 0 <= top_k <= min(MAX_TOP_K, logits.shape[-1]):
        raise RuntimeError(f"top_k must be in [0, min({MAX_TOP_K}, vocab)], got {top_k}")
    if targets.numel() == 0:
        empty = logits.new_empty(lead, dtype=torch.float32) + 0 * logits.sum()
        top = ids = None
        if top_k:
            top, ids = empty[..., None].repeat_interleave(top_k, -1), targets.new_empty(*lead, top_k)
        return TokenLogprobs(empty, empty.clone(), top, ids)
    targets = targets.contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobsFn.apply(logits, targets, top_k, temperature, ignore_index, code))
    rows, at = _as_rows(logits)
    return TokenLogprobs(*_run_logprobs(rows, at, targets, top_k, temperature, ignore_index, code, False)[:4])


class _DistillFn(torch.autograd.Function):
    """fakla_distill_topk with gradients (fakla_distill_topk_backward)."""

    @staticmethod
    def forward(ctx, logits, ids, teacher, lse, temperature, code):
        rows, at = _as_rows(logits)
        loss, stats = _run_distill(rows, at, ids, teacher, lse, temperature, code, True)
        ctx.save_for_backward(rows, ids, teacher, lse, stats)
        ctx.form = at, temperature, code, logits.shape
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        rows, ids, teacher, lse, stats = ctx.saved_tensors
        at, temperature, code, shape = ctx.form
        dloss = dloss.contiguous()
        dlogits = torch.empty_like(rows, memory_format=torch.contiguous_format).view(shape)
        _launch(rows.device, _lib.lib().fakla_distill_topk_backward, _ptr(rows), _ptr(ids), _ptr(teacher), _ptr(lse),
                _ptr(stats), _ptr(dloss), _ptr(dlogits), *at, ids.shape[-1], temperature, code)
        return dlogits, None, None, None, None, None


def _run_distill(rows, at, ids, teacher, lse, temperature, code, save):
    dev = rows.device
    loss = torch.empty(ids.shape[:-1], device=dev, dtype=torch.float32)
    stats = torch.empty((at[0] * at[1], 8), device=dev, dtype=torch.float32) if save else None
    _launch(dev, _lib.lib().fakla_distill_topk, _ptr(rows), _ptr(ids), _ptr(teacher), _ptr(lse), _ptr(loss), _ptr(stats),
            *at, ids.shape[-1], temperature, code)
    return loss, stats


def distill_topk(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                 teacher_lse: Optional[torch.Tensor] = None, *, temperature: float = 1.0) -> torch.Tensor:
    """KL(q || softmax(logits / temperature)) per row, for a teacher q known by
    its largest logits; returns the losses (...) in float32.

    logits: (..., vocab), float32 or bfloat16, read in place as in
    ``token_logprobs``. teacher_ids: (..., K) int64, K up to 256, -1 where a
    row has fewer entries; teacher_logits: (..., K), floating.
    Without ``teacher_lse`` the teacher's distribution is the softmax of its K
    logits / temperature. With it ((...) float: log-sum-exp of the teacher's
    whole row of logits / temperature) the K probabilities are the teacher's
    own, and the mass it gives to all other tokens is compared with the
    model's as one more class.

    A row without entries gives 0 and no gradient. Ids outside of the
    vocabulary (but -1) give NaN and are reported by ``device_status``.
    Differentiable in logits; the teacher's side gets no gradient. The loss is
    not multiplied by temperature squared.
    """
    lead, code, temperature = _check_rows(logits, temperature)
    if teacher_ids.dim() != logits.dim() or teacher_ids.shape != teacher_logits.shape or teacher_ids.shape[:-1] != lead:
        raise RuntimeError(f"teacher_ids {tuple(teacher_ids.shape)} and teacher_logits {tuple(teacher_logits.shape)} "
                           f"must both be (..., K) for logits {tuple(logits.shape)}")
    if teacher_lse is not None and teacher_lse.shape != lead:
        raise RuntimeError(f"teacher_lse {tuple(teacher_lse.shape)} does not go with logits {tuple(logits.shape)}")
    if teacher_ids.dtype != torch.int64:
        raise RuntimeError("teacher_ids must be int64")
    if not teacher_logits.is_floating_point() or (teacher_lse is not None and not teacher_lse.is_floating_point()):
        raise RuntimeError("teacher_logits and teacher_lse must be floating")
    dev = logits.device
    if teacher_ids.device != dev or teacher_logits.device != dev or (teacher_lse is not None and teacher_lse.device != dev):
        raise RuntimeError(f"the teacher's tensors must be on the device of logits ({dev})")
    K = teacher_ids.shape[-1]
    if not 1 <= K <= MAX_ENTRIES:
        raise RuntimeError(f"K must be in [1, {MAX_ENTRIES}], got {K}")
    if teacher_ids.numel() == 0:
        return logits.new_empty(lead, dtype=torch.float32) + 0 * logits.sum()
    ids = teacher_ids.contiguous()
    teacher = teacher_logits.detach().to(torch.float32).contiguous()
    lse = None if teacher_lse is None else teacher_lse.detach().to(torch.float32).contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        return _DistillFn.apply(logits, ids, teacher, lse, temperature, code)
    rows, at = _as_rows(logits)
    return _run_distill(rows, at, ids, teacher, lse, temperature, code, False)[0]
