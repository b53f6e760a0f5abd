"""The language model with recurrent layers trained, distilled and scored: the
recurrence, the token log probabilities and the distillation together, as a
training and scoring program runs them.

Losses are compared with float64 ones of the model's own logits, gradients with
those of the same model whose recurrence is a loop of torch operations and whose
loss is torch's log_softmax. Bars: 1e-4 relative in the 2-norm for fp32
gradients, as for the model's fp32 logits (each kernel stays within 1e-5, and a
gradient passes through a few of them); 3e-2 for bf16 (bf16 activations through
every layer) (GPU only).
"""
import pytest
import torch

from oracle import logits_oracle as O
from tests.helpers import rel_l2, to_np

pytestmark = pytest.mark.gpu

V = 501


def _model(dtype, dev, recurrent=(0, 2)):
    from pulsartecture_b200.lm_harness import FaklaLM

    torch.manual_seed(0)
    return FaklaLM(vocab=V, d_model=128, n_layers=3, n_heads=2, head_dim=64, d_ff=96, n_experts=2, top_k=2,
                   dtype=dtype, recurrent_layers=recurrent).to(dev)


def _ids(B, T, seed=1):
    return torch.randint(0, V, (B, T), generator=torch.Generator().manual_seed(seed))


def _teacher(B, T, K, seed=2):
    full = 2 * torch.randn(B, T, V, generator=torch.Generator().manual_seed(seed))
    top, ids = torch.topk(full, K, dim=-1)
    return ids, top, torch.logsumexp(full, -1)


def _loop(x, gate, state=None, *, gate_act="sigmoid", mix=True, return_state=True):
    a = torch.sigmoid(gate)
    h = torch.zeros_like(x[:, 0]) if state is None else state
    hs = []
    for t in range(x.shape[1]):
        h = a[:, t] * h + (1 - a[:, t]) * x[:, t]
        hs.append(h)
    return torch.stack(hs, 1), h


@pytest.mark.parametrize("dtype,bar", [(torch.float32, 1e-4), (torch.bfloat16, 3e-2)])
def test_losses_scores_and_gradients(cuda, monkeypatch, dtype, bar):
    import pulsartecture_b200.attention.gated_recurrence as R

    B, T, K = 2, 70, 9
    model = _model(dtype, cuda)
    ids = _ids(B, T).to(cuda)
    t_ids, t_top, t_lse = (t.to(cuda) for t in _teacher(B, T, K))
    params = [p for p in model.parameters()]

    loss = model.loss(ids, entropy_weight=0.1)
    distilled = model.distill_loss(ids, t_ids, t_top, t_lse, temperature=1.5)
    logits = model(ids)
    got = torch.autograd.grad(loss + 0.5 * distilled, params)

    targets = torch.cat([ids[:, 1:], torch.full_like(ids[:, :1], -100)], 1)
    want = O.token_logprobs(logits.detach(), targets, 4)
    n = B * (T - 1)
    expected = -(want["logprobs"].sum() + 0.1 * want["entropy"][:, :-1].sum()) / n
    # a mean of values each off by the operators' own bounds, around 1e-6
    assert abs(float(loss.detach()) - float(expected)) <= 1e-5 * (1 + abs(float(expected)))
    expected = O.distill(logits.detach(), t_ids, t_top, t_lse, 1.5)["loss"].mean()
    assert abs(float(distilled.detach()) - float(expected)) <= 1e-5 * (1 + abs(float(expected)))
    r = model.score(ids, top_k=4)
    assert r.logprobs.shape == (B, T - 1) and r.top_ids.shape == (B, T - 1, 4)
    if dtype == torch.float32:
        # (in inference the attention layer folds its projections: other roundings, 1e-4 of the logits)
        assert (r.logprobs.cpu().double() - want["logprobs"][:, :-1]).abs().max() < 1e-2
    assert not r.logprobs.requires_grad

    monkeypatch.setattr(R, "gated_scan", _loop)
    z = model(ids).double()
    lp = torch.log_softmax(z, -1)
    p = lp.exp()
    plain = -(lp[:, :-1].gather(-1, ids[:, 1:, None]).sum() - 0.1 * (p * lp)[:, :-1].sum()) / n
    lt = torch.log_softmax(z / 1.5, -1)
    q = torch.exp(t_top.double() / 1.5 - t_lse.double()[..., None])
    rest_q = (1 - q.sum(-1)).clamp_min(0)
    rest_p = 1 - lt.exp().gather(-1, t_ids).sum(-1)
    kl = (q * (q.log() - lt.gather(-1, t_ids))).sum(-1) + torch.where(rest_q > 0, rest_q * (rest_q.clamp_min(1e-300) / rest_p).log(), 0.0)
    plain = plain + 0.5 * kl.mean()
    exact = torch.autograd.grad(plain, params)
    for (name, _), g, e in zip(model.named_parameters(), got, exact):
        assert torch.isfinite(g).all(), name
        if float(e.double().norm()) > 1e-6 * max(float(x.double().norm()) for x in exact):
            assert rel_l2(to_np(g), to_np(e)) < bar, name


def test_padding_is_left_out(cuda):
    model = _model(torch.float32, cuda, recurrent=(0, 1, 2))
    ids = _ids(2, 30).to(cuda)
    padded = ids.clone()
    padded[1, 20:] = -100
    loss = model.loss(padded)
    # sequence 0 whole and sequence 1 up to its end: the padding behind changes nothing
    a, b = model.loss(ids[:1]), model.loss(ids[1:, :20])
    assert torch.allclose(loss, (29 * a + 19 * b) / 48, rtol=1e-5, atol=1e-6)
    assert float(model.loss(torch.full_like(ids, -100)).detach()) == 0.0
    one = model.loss(ids[:, :1])  # no next token at all
    one.backward()
    assert float(one.detach()) == 0.0


def test_a_captured_training_step_replays(cuda):
    """Loss and gradients of a recurrent layer and the head captured together
    (the mixture of experts reads counts on the host and stays outside)."""
    from pulsartecture_b200 import GatedRecurrence, distill_topk, token_logprobs

    torch.manual_seed(0)
    mixer = GatedRecurrence(64, 96).to(cuda)
    head = torch.nn.Linear(96, V, bias=False).to(cuda)
    params = [*mixer.parameters(), *head.parameters()]
    u = torch.randn(3, 200, 64, device=cuda)
    targets = _ids(3, 200).to(cuda)
    t_ids, t_top, t_lse = (t.to(cuda) for t in _teacher(3, 200, 5))

    def step():
        logits = head(mixer(u))
        r = token_logprobs(logits, targets, top_k=3)
        loss = -r.logprobs.mean() - 0.01 * r.entropy.mean() + distill_topk(logits, t_ids, t_top, t_lse).mean()
        return [loss.detach(), r.top_ids, *torch.autograd.grad(loss, params)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (5, 6):
        u.copy_(torch.randn(3, 200, 64, generator=torch.Generator().manual_seed(seed)).to(cuda))
        targets.copy_(_ids(3, 200, seed).to(cuda))
        graph.replay()
        for a, b in zip(held, step()):
            if a.dtype == torch.int64:
                assert torch.equal(a, b)
            else:  # the library products of a capture may run another algorithm
                assert rel_l2(to_np(a), to_np(b)) < 1e-5


def test_calls_on_two_streams_at_once(cuda):
    from pulsartecture_b200 import gated_scan, token_logprobs

    def work(seed):
        g = torch.Generator(device=cuda).manual_seed(seed)
        x, gate = (torch.randn(4, 3000, 256, generator=g, device=cuda).bfloat16() for _ in range(2))
        z = torch.randn(300, 20011, generator=g, device=cuda)
        t = torch.randint(0, 20011, (300,), generator=g, device=cuda)
        torch.cuda.current_stream().synchronize()
        return lambda: (*gated_scan(x, gate), *token_logprobs(z, t, top_k=7))

    streams = [torch.cuda.Stream() for _ in range(2)]
    jobs = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            jobs.append(work(i))
    alone = []
    for j, s in zip(jobs, streams):
        with torch.cuda.stream(s):
            alone.append(j())
        torch.cuda.synchronize()
    together = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                together[i].append(jobs[i]())
    torch.cuda.synchronize()
    for i in range(2):
        for got in together[i]:
            for a, b in zip(got, alone[i]):
                assert torch.equal(a, b)
