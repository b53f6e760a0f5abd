"""float64 restatement of the operators on rows of logits: token log
probabilities with entropies and the largest entries, and the divergence from
a teacher's largest logits. Gradients come from the formulas, written out."""
from __future__ import annotations

import math

import torch


def log_softmax(z: torch.Tensor) -> torch.Tensor:
    """Over the last dimension; a row of nothing but -inf gives -inf."""
    m = z.amax(-1, keepdim=True)
    z = z - torch.where(m == -math.inf, torch.zeros_like(m), m)
    s = torch.exp(z).sum(-1, keepdim=True)
    return z - torch.where(s == 0, torch.zeros_like(s), torch.log(s))


def _times(p, v):
    """p v, with 0 wherever p is 0."""
    return torch.where(p == 0, torch.zeros_like(p), p * v)


def token_logprobs(logits, targets, top_k=0, temperature=1.0, ignore_index=-100, dlp=None, dent=None, dtop=None):
    x = logits.double().cpu()
    targets = targets.cpu()
    # the difference first: values near the end of a type's range stay finite
    m = x.amax(-1, keepdim=True)
    lp = log_softmax((x - torch.where(torch.isinf(m), torch.zeros_like(m), m)) / temperature)
    p = torch.exp(lp)
    counted = targets != ignore_index
    at = torch.where(counted, targets, 0)[..., None]
    got = {"logprobs": torch.where(counted, lp.gather(-1, at)[..., 0], 0.0),
           "entropy": -_times(p, lp).sum(-1), "p": p, "lp": lp}
    if top_k:
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top_k]
        got["top_ids"], got["top_logprobs"] = ids, lp.gather(-1, ids)
    if dlp is not None or dent is not None or dtop is not None:
        dz = torch.zeros_like(p)
        if dlp is not None:
            w = torch.where(counted, dlp.double().cpu(), 0.0)[..., None]
            dz -= p * w
            dz.scatter_add_(-1, at, w)
        if dent is not None:
            dz -= dent.double().cpu()[..., None] * _times(p, lp + got["entropy"][..., None])
        if dtop is not None:
            d = dtop.double().cpu()
            dz -= p * d.sum(-1, keepdim=True)
            dz.scatter_add_(-1, got["top_ids"], d)
        empty = (x == -math.inf).all(-1, keepdim=True)
        got["dlogits"] = torch.where(empty, 0.0, dz / temperature)
    return got


def distill(logits, ids, teacher, lse=None, temperature=1.0, dloss=None):
    x = logits.double().cpu().reshape(-1, logits.shape[-1])
    K = ids.shape[-1]
    ids, t = ids.cpu().reshape(-1, K), teacher.double().cpu().reshape(-1, K) / temperature
    lp = log_softmax(x / temperature)
    p = torch.exp(lp)
    loss, dz = torch.zeros(len(x), dtype=torch.float64), torch.zeros_like(x)
    for r in range(len(x)):
        keep = ids[r] >= 0
        i, tr = ids[r][keep], t[r][keep]
        if not len(i) or (lse is None and torch.all(tr == -math.inf)):
            continue
        lq = tr - lse.double().cpu().reshape(-1)[r] if lse is not None else tr - torch.logsumexp(tr, 0)
        q = torch.exp(lq)
        loss[r] = _times(q, lq - lp[r][i]).sum()
        mass = q.sum()
        rest = torch.ones_like(p[r])
        if lse is not None:
            rest[i] = 0
            qr = max(0.0, 1.0 - float(mass))
            pr = (p[r] * rest).sum()
            if qr > 0:
                loss[r] += qr * (math.log(qr) - torch.log(pr))
                dz[r] -= _times(p[r] * rest, qr / pr)
            mass = mass + qr
        dz[r] += p[r] * mass
        if torch.any(torch.isfinite(x[r])):
            dz[r].index_add_(0, i, -q)
    got = {"loss": loss.reshape(logits.shape[:-1]), "p": p.reshape(logits.shape)}
    if dloss is not None:
        g = dloss.double().cpu().reshape(-1, 1) / temperature
        got["dlogits"] = (dz * g).reshape(logits.shape)
    return got
