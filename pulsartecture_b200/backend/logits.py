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
from .interface import _check_device, _dtype_code, _needs_grad, _ptr, _require, _stream

MAX_TOP_K = 32
MAX_ENTRIES = 256


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor                 # (...) float32
    entropy: torch.Tensor                  # (...) float32
    top_logprobs: Optional[torch.Tensor]   # (..., top_k) float32, or None
    top_ids: Optional[torch.Tensor]        # (..., top_k) int64, or None


def _as_rows(logits: torch.Tensor) -> torch.Tensor:
    """(batch, rows, vocab) over the same values: a view wherever the leading
    dimensions come down to two strides (a slice of positions or a padded
    vocabulary does), a dense copy otherwise."""
    if logits.stride(-1) != 1 and logits.shape[-1] != 1:
        logits = logits.contiguous()
    if logits.dim() == 3:
        return logits
    if logits.dim() < 3:
        return logits.reshape(1, -1, logits.shape[-1])
    return logits.reshape(-1, *logits.shape[-2:])


def _check_rows(logits: torch.Tensor, given, names, lead_of) -> torch.device:
    _require(logits.dim() >= 1 and logits.shape[-1] >= 1, "logits must be (..., vocab)")
    dev = _check_device([logits, *given], ["logits", *names])
    lead = tuple(logits.shape[:-1])
    for t, n in zip(given, names):
        if t is not None:
            got = tuple(t.shape[:len(lead)]) if n in lead_of else tuple(t.shape)
            _require(got == lead, f"{n} {tuple(t.shape)} does not go with logits {tuple(logits.shape)}")
    return dev


def _check_temperature(temperature: float) -> float:
    temperature = float(temperature)
    _require(1e-30 <= temperature <= 1e30, f"temperature must be positive (1e-30 to 1e30), got {temperature}")
    return temperature


class _TokenLogprobsFn(torch.autograd.Function):
    """fakla_token_logprobs with gradients (fakla_token_logprobs_backward)."""

    @staticmethod
    def forward(ctx, logits, targets, top_k, temperature, ignore_index):
        ctx.set_materialize_grads(False)
        lp, ent, top, ids, stats = _run_logprobs(logits, targets, top_k, temperature, ignore_index, True)
        ctx.save_for_backward(logits, targets, stats, ent, ids)
        ctx.top_k, ctx.temperature, ctx.ignore_index = top_k, temperature, ignore_index
        if top_k:
            ctx.mark_non_differentiable(ids)
        return lp, ent, top, ids

    @staticmethod
    @once_differentiable
    def backward(ctx, dlp, dent, dtop, _):
        logits, targets, stats, ent, ids = ctx.saved_tensors
        dlp, dent, dtop = (None if t is None else t.contiguous().float() for t in (dlp, dent, dtop))
        dlogits = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
        dev = logits.device
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().fakla_token_logprobs_backward(
                _ptr(logits), _ptr(targets), _ptr(stats), _ptr(ent), _ptr(ids), _ptr(dlp), _ptr(dent), _ptr(dtop),
                _ptr(dlogits), *logits.shape, logits.stride(0), logits.stride(1), ctx.top_k, ctx.temperature,
                ctx.ignore_index, _dtype_code(logits), _stream(dev)))
        return dlogits, None, None, None, None


def _run_logprobs(logits, targets, top_k, temperature, ignore_index, save):
    """logits (batch, rows, vocab); everything it returns is (batch, rows, ...)."""
    dev = logits.device
    lead = logits.shape[:2]
    lp = torch.empty(lead, device=dev, dtype=torch.float32)
    ent = torch.empty(lead, device=dev, dtype=torch.float32)
    top = torch.empty(*lead, top_k, device=dev, dtype=torch.float32) if top_k else None
    ids = torch.empty(*lead, top_k, device=dev, dtype=torch.int64) if top_k else None
    stats = torch.empty(*lead, 2, device=dev, dtype=torch.float32) if save else None
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().fakla_token_logprobs(
            _ptr(logits), _ptr(targets), _ptr(lp), _ptr(ent), _ptr(top), _ptr(ids), _ptr(stats), *logits.shape,
            logits.stride(0), logits.stride(1), top_k, temperature, ignore_index, _dtype_code(logits), _stream(dev)))
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
    temperature = _check_temperature(temperature)
    _check_rows(logits, [targets], ["targets"], ())
    _require(targets.dtype == torch.int64, "targets must be int64")
    V = logits.shape[-1]
    _require(0 <= top_k <= min(MAX_TOP_K, V), f"top_k must be in [0, min({MAX_TOP_K}, vocab)], got {top_k}")
    _dtype_code(logits)
    lead = logits.shape[:-1]
    if targets.numel() == 0:
        empty = logits.new_empty(lead, dtype=torch.float32) + 0 * logits.sum()
        top = ids = None
        if top_k:
            top, ids = logits.new_empty(*lead, top_k, dtype=torch.float32), targets.new_empty(*lead, top_k)
        return TokenLogprobs(empty, empty.clone(), top, ids)
    rows = _as_rows(logits)
    flat = targets.contiguous()
    if _needs_grad(logits):
        lp, ent, top, ids = _TokenLogprobsFn.apply(rows, flat, top_k, temperature, ignore_index)
    else:
        lp, ent, top, ids, _ = _run_logprobs(rows, flat, top_k, temperature, ignore_index, False)
    if top_k:
        top, ids = top.reshape(*lead, top_k), ids.reshape(*lead, top_k)
    return TokenLogprobs(lp.reshape(lead), ent.reshape(lead), top, ids)


class _DistillFn(torch.autograd.Function):
    """fakla_distill_topk with gradients (fakla_distill_topk_backward)."""

    @staticmethod
    def forward(ctx, logits, ids, teacher, lse, temperature):
        loss, stats = _run_distill(logits, ids, teacher, lse, temperature, True)
        ctx.save_for_backward(logits, ids, teacher, lse, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        logits, ids, teacher, lse, stats = ctx.saved_tensors
        dloss = dloss.contiguous().float()
        dlogits = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
        dev = logits.device
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().fakla_distill_topk_backward(
                _ptr(logits), _ptr(ids), _ptr(teacher), _ptr(lse), _ptr(stats), _ptr(dloss), _ptr(dlogits),
                *logits.shape, logits.stride(0), logits.stride(1), ids.shape[-1], ctx.temperature,
                _dtype_code(logits), _stream(dev)))
        return dlogits, None, None, None, None


def _run_distill(logits, ids, teacher, lse, temperature, save):
    dev = logits.device
    loss = torch.empty(logits.shape[:2], device=dev, dtype=torch.float32)
    stats = torch.empty(*logits.shape[:2], 8, device=dev, dtype=torch.float32) if save else None
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().fakla_distill_topk(
            _ptr(logits), _ptr(ids), _ptr(teacher), _ptr(lse), _ptr(loss), _ptr(stats), *logits.shape,
            logits.stride(0), logits.stride(1), ids.shape[-1], temperature, _dtype_code(logits), _stream(dev)))
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
    temperature = _check_temperature(temperature)
    _check_rows(logits, [teacher_ids, teacher_logits, teacher_lse], ["teacher_ids", "teacher_logits", "teacher_lse"],
                ("teacher_ids", "teacher_logits"))
    lead = logits.shape[:-1]
    _require(teacher_ids.dim() == logits.dim() and teacher_ids.shape == teacher_logits.shape,
             "teacher_ids and teacher_logits must both be (..., K)")
    _require(teacher_ids.dtype == torch.int64, "teacher_ids must be int64")
    _require(teacher_logits.is_floating_point() and (teacher_lse is None or teacher_lse.is_floating_point()),
             "teacher_logits and teacher_lse must be floating")
    K = teacher_ids.shape[-1]
    _require(1 <= K <= MAX_ENTRIES, f"K must be in [1, {MAX_ENTRIES}], got {K}")
    _dtype_code(logits)
    if teacher_ids.numel() == 0:
        return logits.new_empty(lead, dtype=torch.float32) + 0 * logits.sum()
    rows = _as_rows(logits)
    ids = teacher_ids.contiguous()
    teacher = teacher_logits.detach().float().contiguous()
    lse = None if teacher_lse is None else teacher_lse.detach().float().contiguous()
    if _needs_grad(logits):
        loss = _DistillFn.apply(rows, ids, teacher, lse, temperature)
    else:
        loss, _ = _run_distill(rows, ids, teacher, lse, temperature, False)
    return loss.reshape(lead)
