"""Padded batches in the language model's scoring and distillation, with the
operators and the layers replaced by float64 stand-ins. CPU only."""
import pytest
import torch

from oracle import logits_oracle as O
from pulsartecture_b200 import lm_harness
from pulsartecture_b200.backend.logits import TokenLogprobs

V = 31


@pytest.fixture
def model(monkeypatch):
    torch.manual_seed(0)
    m = lm_harness.FaklaLM(vocab=V, d_model=8, n_layers=1, n_heads=1, head_dim=64, d_ff=8, n_experts=1, top_k=1)
    m = m.double()
    monkeypatch.setattr(m, "forward", lambda ids: m.head(m.embed(ids)))

    def distill(logits, ids, teacher, lse=None, *, temperature=1.0):
        return O.distill(logits.detach(), ids, teacher, lse, temperature)["loss"]

    def score(logits, targets, *, top_k=0, temperature=1.0, ignore_index=-100):
        r = O.token_logprobs(logits.detach(), targets, top_k, temperature, ignore_index)
        return TokenLogprobs(r["logprobs"], r["entropy"], r.get("top_logprobs"), r.get("top_ids"))

    monkeypatch.setattr(lm_harness, "distill_topk", distill)
    monkeypatch.setattr(lm_harness, "token_logprobs", score)
    return m


def _batch(B=3, T=12, K=4):
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, V, (B, T), generator=g)
    full = torch.randn(B, T, V, generator=g, dtype=torch.float64)
    top, t_ids = torch.topk(full, K, dim=-1)
    return ids, t_ids, top, torch.logsumexp(full, -1)


@pytest.mark.parametrize("rest", [False, True])
def test_positions_without_a_teacher_do_not_count(model, rest):
    """A mean over the positions that have an entry; 0 where none has."""
    ids, t_ids, top, lse = _batch()
    lse = lse if rest else None
    whole = model.distill_loss(ids, t_ids, top, lse)
    per = lm_harness.distill_topk(model(ids), t_ids, top, lse)
    assert abs(float(whole - per.mean())) < 1e-12
    t_ids[1, 7:] = -1
    t_ids[2] = -1
    t_ids[0, 3, 1:] = -1  # fewer entries, but some
    per = lm_harness.distill_topk(model(ids), t_ids, top, lse)
    got = model.distill_loss(ids, t_ids, top, lse)
    assert abs(float(got - per.sum() / (12 + 7))) < 1e-12
    assert float(model.distill_loss(ids, torch.full_like(t_ids, -1), top, lse)) == 0.0


def test_padded_ids_are_not_embedded(model):
    """Padding (ignore_index) in score and distill_loss, as in loss."""
    ids, t_ids, top, lse = _batch()
    padded = ids.clone()
    padded[1, 7:] = -100
    padded[2, :] = -100
    r, w = model.score(padded, top_k=2), model.score(ids, top_k=2)
    assert r.logprobs.shape == (3, 11) and r.top_ids.shape == (3, 11, 2)
    assert torch.equal(r.logprobs[0], w.logprobs[0]) and torch.equal(r.logprobs[1, :6], w.logprobs[1, :6])
    assert not r.logprobs[1, 6:].any() and not r.logprobs[2].any()
    got = model.distill_loss(padded, t_ids, top, lse)
    per = lm_harness.distill_topk(model(ids), t_ids, top, lse)
    assert abs(float(got - (per[0].sum() + per[1, :7].sum()) / 19)) < 1e-12
    # another mark, which is a token of the vocabulary
    marked = ids.clone()
    marked[0, 9:] = 5
    a = model.score(marked, ignore_index=5)
    assert not a.logprobs[0, 8:].any()
    assert float(model.distill_loss(torch.full_like(ids, -7), t_ids, top, ignore_index=-7)) == 0.0
