"""A padded batch scored and distilled: as its sequences without the padding
(GPU only). Sequences go through other launches there, whose sums may run in
another order: bars as for the model's padded loss."""
import pytest
import torch

from tests.test_gpu_lm_training import _ids, _model, _teacher

pytestmark = pytest.mark.gpu


def test_padded_batch(cuda):
    model = _model(torch.float32, cuda, recurrent=(0, 1, 2))
    ids = _ids(2, 30).to(cuda)
    t_ids, t_top, t_lse = (t.to(cuda) for t in _teacher(2, 30, 6))
    padded = ids.clone()
    padded[1, 20:] = -100
    r = model.score(padded, top_k=2)
    for row, n in ((0, 29), (1, 19)):
        w = model.score(ids[row:row + 1, :n + 1], top_k=2)
        assert torch.allclose(r.logprobs[row, :n], w.logprobs[0], rtol=1e-5, atol=1e-5)
        assert torch.allclose(r.entropy[row, :n], w.entropy[0], rtol=1e-5, atol=1e-5)
        assert torch.equal(r.top_ids[row, :n], w.top_ids[0])
    assert not r.logprobs[1, 19:].any()
    for lse in (None, t_lse):
        loss = model.distill_loss(padded, t_ids, t_top, lse)
        cut = lambda t, row, n: None if t is None else t[row:row + 1, :n]  # noqa: E731
        parts = [n * model.distill_loss(*(cut(t, row, n) for t in (ids, t_ids, t_top, lse))) for row, n in ((0, 30), (1, 20))]
        assert torch.allclose(loss, sum(parts) / 50, rtol=1e-5, atol=1e-6)
        grads = torch.autograd.grad(loss, [p for p in model.parameters()], allow_unused=True)
        assert all(g is None or torch.isfinite(g).all() for g in grads)
