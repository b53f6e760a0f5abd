"""Rows of logits at the edges of their definition: rows that are given
nothing, rows without a distribution behind them, a model that leaves next to
nothing outside of the teacher's entries, temperatures close to 0, repeated
entries, calls from two threads.

Bounds as in test_gpu_logits.py, u = 2^-24 (GPU only).
"""
import threading

import pytest
import torch

from tests.test_gpu_logits import INF, U, _check_token, _logits, _sum_error, _teacher, _within

pytestmark = pytest.mark.gpu

NAN = float("nan")
TYPES = [torch.float32, torch.bfloat16]
# 5003 values: rows start and end on no 16 bytes, in either type


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rest", [False, True])
def test_distill_rows_given_zero(cuda, dtype, rest):
    """A row whose loss counts for nothing gets no gradient whatever it holds:
    a bad id, a NaN or +inf, nothing but -inf, values far from 0."""
    from pulsartecture_b200 import _lib, distill_topk
    from pulsartecture_b200.backend.interface import device_status

    device_status()
    for V in (5003, 40001):
        rows, K = 14, 6
        ids, top, lse, full = _teacher((rows,), V, K, V, 1.0)
        logits = full.to(dtype)
        ids[0:2, 2] = V
        ids[2:4, 1] = -100
        logits[4:6, 7] = NAN
        logits[6:8, 9] = INF
        logits[8:10] = -INF
        logits[10:12] += 3e6  # past where the kernels form their exponents by one product
        ids[11, 3] = V + 5
        given = torch.zeros(rows)
        given[12:] = 1.5
        leaf = logits.to(cuda).requires_grad_()
        loss = distill_topk(leaf, ids.to(cuda), top.to(cuda), lse.to(cuda) if rest else None)
        assert torch.isnan(loss[[0, 1, 2, 3, 4, 5, 6, 7, 11]]).all() and (loss[8:10] == INF).all()
        g, = torch.autograd.grad(loss, leaf, given.to(cuda))
        assert not torch.isnan(g).any() and not g[:12].any()
        assert torch.isfinite(g[12:]).all() and g[12:].any()
        with pytest.raises(_lib.FaklaError):
            device_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rest", [False, True])
def test_distill_rows_without_entries(cuda, dtype, rest):
    """No entry: loss 0 and no gradient, whatever the row's logits are."""
    from pulsartecture_b200 import distill_topk

    for V in (5003, 40001):
        rows, K = 7, 6
        ids, top, lse, full = _teacher((rows,), V, K, V, 1.0)
        logits = full.to(dtype)
        logits[0, 7] = logits[1, V - 1] = NAN
        logits[2, 0] = INF
        logits[3] = -INF
        logits[4] = -3e6
        ids[:6] = -1
        top[5] = NAN  # nothing is read where there is no entry
        leaf = logits.to(cuda).requires_grad_()
        loss = distill_topk(leaf, ids.to(cuda), top.to(cuda), lse.to(cuda) if rest else None)
        g, = torch.autograd.grad(loss.sum(), leaf)
        assert not loss[:6].any() and not torch.isnan(loss).any() and loss[6] != 0
        assert not torch.isnan(g).any() and not g[:6].any() and g[6].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top_k", [0, 3])
def test_token_rows_given_zero(cuda, dtype, top_k):
    """A row that is given only zeros (an ignored target's log probability
    counts as that) gets no gradient: one with a NaN, one with +inf, one with a
    target outside of the vocabulary. Given anything, it gets NaN."""
    from pulsartecture_b200 import _lib, token_logprobs
    from pulsartecture_b200.backend.interface import device_status

    device_status()
    for V in (5003, 40001):
        logits = _logits((12,), V, dtype)
        logits[0:3, 11] = NAN
        logits[3:6, V - 1] = INF
        targets = torch.full((12,), 5)
        targets[1] = targets[4] = -100
        targets[6:8] = V
        given = torch.zeros(12)
        given[1] = given[4] = 2.0  # ignored
        given[2] = given[5] = given[7] = given[10] = 2.0
        leaf = logits.to(cuda).requires_grad_()
        r = token_logprobs(leaf, targets.to(cuda), top_k=top_k)
        zeros = torch.zeros(12, device=cuda)
        for outs, grads in (([r.logprobs], [given]), ([r.logprobs, r.entropy], [given, zeros]),
                            ([r.logprobs, r.entropy, r.top_logprobs], [given, zeros, torch.zeros(12, top_k)])):
            if outs[-1] is None:
                continue
            g, = torch.autograd.grad(outs, leaf, [t.to(cuda) for t in grads], retain_graph=True)
            nan = torch.isnan(g)
            for row in (2, 5, 7):
                assert nan[row].all(), row
            for row in (0, 1, 3, 4, 6, 8, 9, 11):
                assert not nan[row].any() and not g[row].any(), row
            assert torch.isfinite(g[10]).all() and g[10].any()
        # the entropy's gradient does not depend on the target
        g, = torch.autograd.grad(r.entropy, leaf, torch.ones(12, device=cuda))
        assert torch.isnan(g).any(1).tolist() == [True] * 6 + [False] * 6 and g[6].any()
        with pytest.raises(_lib.FaklaError):
            device_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1e-30, 1e-9, 1e-4, 1e30])
def test_extreme_temperatures(cuda, dtype, temperature):
    """All three gradients where softmax is a maximum, or flat; masked places
    get 0. Some rows have two largest values, some their maximum at 0."""
    V = 5003
    logits = _logits((6,), V, dtype)
    logits[1, ::3] = -INF
    logits[2, 1::2] = -INF
    top = logits[2].max() + 1
    logits[2, [0, 4000]] = top
    logits[3] -= logits[3].max()
    logits[4] -= logits[4].max()
    logits[4, 2500:] = -INF
    logits[5, :] = -INF
    logits[5, V - 1] = 1.0
    targets = torch.tensor([7, 0, 4000, 5, 3000, V - 1])
    _check_token(cuda, logits, targets, 2, temperature)


def _check_rest(cuda, logits, ids, teacher, lse, temperature):
    """Loss and gradient with the rest as a class, in logarithms throughout.

    Outside of the entries a gradient is p_j (Q + q_r) - q_r p_j / p_r. Both
    terms go by their own size: p_j is off by 8 u of its logarithm and by what
    its sum is off by (`err`), q_r by K u and the q's own errors, and p_j / p_r by
    8 u of the distance d to the largest logit outside, where p_r is summed on its
    own; where it is 1 less the entries' sum, p_r is at least q_r / 4 > 10^-4.6
    and |log p_j| at most d + 11 + log V < d + 24."""
    from pulsartecture_b200 import distill_topk

    V = logits.shape[-1]
    x = logits.double()
    y = (x - x.amax(-1, keepdim=True)) / temperature
    total = torch.logsumexp(y, -1, keepdim=True)
    lp = y - total
    lq = teacher.double() / temperature - lse.double()[:, None]
    q = torch.exp(lq)
    out = torch.ones_like(x, dtype=torch.bool).scatter_(-1, ids, False)
    most_out = torch.where(out, x, -INF).amax(-1, keepdim=True)
    below = torch.where(out, (x - most_out) / temperature, -INF)
    sum_out = torch.logsumexp(below, -1, keepdim=True)
    lpr = ((most_out - x.amax(-1, keepdim=True)) / temperature - total + sum_out)[:, 0]
    qr = (1 - q.sum(-1)).clamp_min(0)
    assert (qr > 1e-4).all()
    given = torch.randn(len(x), generator=torch.Generator().manual_seed(9))
    at = lp.gather(-1, ids)
    want = (q * (lq - at)).sum(-1) + qr * (qr.log() - lpr)
    leaf = logits.to(cuda).requires_grad_()
    loss = distill_topk(leaf, ids.to(cuda), teacher.to(cuda), lse.to(cuda), temperature=temperature)
    g, = torch.autograd.grad(loss, leaf, given.to(cuda))

    p = torch.exp(lp)
    err = _sum_error(V, lp, p)
    size = teacher.double().abs().amax(-1) / temperature + lse.double().abs()
    qerr = U * (8 + 4 * size + 2 * ids.shape[-1])
    gap = 1 + torch.maximum(at.abs().amax(-1), lpr.abs())
    _within(loss, want, (qerr * gap + 2 * err + 8 * U * gap) * 2, "loss")
    c = (given.double() / temperature)[:, None]
    ratio = torch.exp(below - sum_out)
    one, two = p * (q.sum(-1) + qr)[:, None], qr[:, None] * ratio
    value = c * torch.where(out, one - two, one - torch.zeros_like(p).scatter_add_(-1, ids, q))
    d = torch.where(ratio > 0, -below, 0.0)
    size_p = torch.where(p > 0, lp.abs(), 0.0)
    most = one * (err[:, None] + 8 * U * (size_p + 24)) + two * (err[:, None] + U * (V / 128 + 40) + 8 * U * (d + 24))
    most = most + qerr[:, None] * (p + ratio)
    most.scatter_add_(-1, ids, (qerr[:, None] + 8 * U) * q)
    # results and terms below 2^-126 flush to 0
    _within(g, value, c.abs() * (most + 2.0 ** -125) + 4 * U * value.abs(), "dlogits")
    return loss


@pytest.mark.parametrize("rows,V", [(3, 40001), (200, 1000)])
@pytest.mark.parametrize("scale", [1.0, 8.0, 20.0, 25.0, 40.0, 100.0, 1000.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_next_to_nothing_outside(cuda, rows, V, scale, dtype):
    """The model's mass outside of the entries from its ordinary size down to
    far below the smallest fp32 number: a finite loss, and a gradient there
    that goes by what the teacher leaves."""
    ids, top, lse, full = _teacher((rows,), V, 40, 5, 1.0)
    assert torch.isfinite(_check_rest(cuda, (full * scale).to(dtype), ids, top, lse, 1.0)).all()


@pytest.mark.parametrize("offset", [2e6, -3e6])
def test_distill_next_to_nothing_outside_far_from_zero(cuda, offset):
    for rows, V in ((3, 40001), (200, 1000)):
        ids, top, lse, full = _teacher((rows,), V, 40, 5, 1.0)
        _check_rest(cuda, full * 40 + offset, ids, top, lse, 1.0)


def test_distill_some_of_the_rest_masked(cuda):
    """Outside logits of -inf beside others far below the entries; then all of
    them masked, by the type's lowest value and by -inf."""
    from pulsartecture_b200 import distill_topk

    V = 5003
    ids, top, lse, full = _teacher((4,), V, 40, 5, 1.0)
    logits = full * 40
    out = torch.ones(4, V, dtype=torch.bool).scatter_(-1, ids, False)
    logits[out & (torch.arange(V) % 3 > 0)] = -INF
    _check_rest(cuda, logits, ids, top, lse, 1.0)
    for dtype in TYPES:
        for mask in (torch.finfo(dtype).min, -INF):
            masked = logits.to(dtype)
            masked[out] = mask
            leaf = masked.to(cuda).requires_grad_()
            loss = distill_topk(leaf, ids.to(cuda), top.to(cuda), lse.to(cuda))
            g, = torch.autograd.grad(loss.sum(), leaf)
            assert (loss == INF).all() and torch.isfinite(g).all() and not g.cpu()[out].any()


@pytest.mark.parametrize("V,K", [(33, 7), (1000, 64), (4099, 200), (32000, 50), (50257, 17)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_distill_rest_gradient(cuda, V, K, dtype, temperature):
    """The gradient of every logit outside of the entries by its own size."""
    ids, top, lse, full = _teacher((6,), V, K, V + K, temperature)
    logits = (full * 0.7 + torch.randn(6, V, generator=torch.Generator().manual_seed(K))).to(dtype)
    _check_rest(cuda, logits, ids, top, lse, temperature)


@pytest.mark.parametrize("rows,V", [(6, 40000), (3000, 2000)])  # (rows start alike on 16 bytes)
def test_distill_repeated_entries_are_the_same_bits(cuda, rows, V):
    """Rows that are all alike, with ids named by several warps' threads, most
    of the model's mass at them and a small divergence: one loss and one
    gradient, on every row and every run."""
    from pulsartecture_b200 import distill_topk

    g = torch.Generator().manual_seed(1)
    K = 256
    full = torch.randn(V, generator=g)
    ids = torch.randint(0, 90, (K,), generator=g) * (V // 91)
    full[ids] += 8.0
    logits = full.expand(rows, V).contiguous().to(cuda).requires_grad_()
    top = full[ids] + 0.2 * torch.randn(K, generator=g)
    lse = torch.logsumexp(top, 0) + 0.2
    args = [ids.expand(rows, K).to(cuda), top.expand(rows, K).to(cuda), lse.expand(rows).to(cuda)]
    first = None
    for _ in range(20):
        loss = distill_topk(logits, *args)
        grad, = torch.autograd.grad(loss.sum(), logits)
        if first is None:
            first = loss[0].item(), grad[0].clone()
        assert (loss == first[0]).all()
        assert (grad == first[1]).all()


def test_alternatives_from_two_threads(cuda):
    """Vocabularies that ask for different amounts of shared memory, scored by
    two threads at once: each call is as valid as alone."""
    from pulsartecture_b200 import _lib, token_logprobs

    errors, found = [], {}
    start = threading.Barrier(2)

    def work(V):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                logits = torch.zeros(1, V, device=cuda)
                logits[:, 9] = 1.0
                targets = torch.zeros(1, dtype=torch.int64, device=cuda)
                r = token_logprobs(logits, targets, top_k=2)
                stream.synchronize()
                call = _lib.lib().fakla_token_logprobs
                args = [t.data_ptr() for t in (logits, targets, r.logprobs, r.entropy, r.top_logprobs, r.top_ids)]
                args += [None, 1, 1, V, V, V, 2, 1.0, -100, _lib.FAKLA_F32, stream.cuda_stream]
                start.wait(60)
                for _ in range(20000):
                    _lib.check(call(*args))
                stream.synchronize()
                found[V] = r.top_ids.tolist()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    sizes = (270000, 1000000)
    threads = [threading.Thread(target=work, args=(V,)) for V in sizes]
    for t in threads:
        t.start()
    for t in threads:
        t.join(300)
    assert not errors, errors[0]
    assert all(found[V] == [[9, 0]] for V in sizes)
