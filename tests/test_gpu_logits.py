"""token_logprobs and distill_topk against the float64 restatement
(oracle/logits_oracle.py).

Bounds, with u = 2^-24 and d = |x - max| / temperature: a term e^{-d} is off by
4u (the exponential) + 3 d u (its argument), so a weight p by that and what the
sum is off by; adding up to V terms over 128 or more threads is off by at most
(V / 128 + 16) u, and the terms' own errors average to (4 + 3 sum p d) u. log s
and log p are off by that much, absolutely, plus a rounding of their own value.
Storing bf16 gradients adds half a step, 2^-8 of the value (GPU only).
"""
import math

import pytest
import torch

from oracle import logits_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = math.inf


def _sum_error(V, lp, p):
    """How far log s, and so each log p beside its own rounding, may be off: (...,)."""
    d = torch.where(p == 0, 0.0, lp.amax(-1, keepdim=True) - lp)
    return U * (V / 128 + 24 + 4 * (p * d).sum(-1))


def _within(got, value, tol, name):
    got = got.detach().cpu()
    step = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    value, tol = value.expand(got.shape), tol.expand(got.shape)
    past = value.abs() > torch.finfo(torch.float32).max  # -3.4e38 / 0.5 is -inf in 32 bits
    value = torch.where(past, torch.sign(value) * INF, value)
    finite = torch.isfinite(value)
    assert torch.equal(torch.isnan(got), torch.isnan(value)), name
    assert torch.equal(got.double()[~finite].nan_to_num(7.0), value[~finite].nan_to_num(7.0)), name
    off = (got.double() - value)[finite].abs()
    most = (tol + step * (value.abs() + tol) + 2.0 ** -126)[finite]
    assert bool((off <= most).all()), (name, float((off / most).max()))


def _logits(rows, V, dtype, seed=0, scale=3.0):
    return (torch.randn(*rows, V, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _check_token(cuda, logits, targets, top_k, temperature, ignore_index=-100, grads=True, on=None, seed=1):
    """logits on the CPU (the values); `on`: the tensor of the device to call with."""
    from pulsartecture_b200 import token_logprobs

    V = logits.shape[-1]
    lead = logits.shape[:-1]
    g = torch.Generator().manual_seed(seed)
    dlp, dent = torch.randn(lead, generator=g), torch.randn(lead, generator=g)
    dtop = torch.randn(*lead, top_k, generator=g) if top_k else None
    want = O.token_logprobs(logits, targets, top_k, temperature, ignore_index, dlp, dent, dtop)
    on = logits.to(cuda) if on is None else on
    leaf = on.detach().requires_grad_(grads)
    r = token_logprobs(leaf, targets.to(cuda), top_k=top_k, temperature=temperature, ignore_index=ignore_index)
    assert r.logprobs.shape == lead and r.entropy.shape == lead
    err = _sum_error(V, want["lp"], want["p"])
    own = lambda v: 3 * U * torch.where(torch.isfinite(v), v.abs(), 0.0)  # noqa: E731
    _within(r.logprobs, want["logprobs"], err + own(want["logprobs"]) * 2, "logprobs")
    H = want["entropy"]
    _within(r.entropy, H, 3 * err * (1 + H.abs()), "entropy")
    if top_k:
        assert torch.equal(r.top_ids.cpu(), want["top_ids"])
        _within(r.top_logprobs, want["top_logprobs"], err[..., None] + own(want["top_logprobs"]) * 2, "top_logprobs")
    if grads:
        outs, given = [r.logprobs, r.entropy], [dlp, dent]
        if top_k:
            outs, given = outs + [r.top_logprobs], given + [dtop]
        got, = torch.autograd.grad(outs, leaf, [t.to(cuda) for t in given])
        assert got.dtype == leaf.dtype and got.shape == leaf.shape
        p, lp = want["p"], want["lp"]
        lpz = torch.where(p == 0, 0.0, lp)
        rel = err[..., None] + U * (8 + 4 * lpz.abs())
        w = torch.where(targets != ignore_index, dlp.double(), 0.0).abs() + (dtop.double().abs().sum(-1) if top_k else 0)
        size = p * (w[..., None] + dent.double().abs()[..., None] * (lpz.abs() + H.abs()[..., None]))
        size2 = p * dent.double().abs()[..., None] * (3 * err * (1 + H.abs()))[..., None]
        most = (size * (rel + 4 * U) + size2) / temperature + 4 * U * want["dlogits"].abs()
        # entries of a target or an alternative also hold its gradient itself
        if top_k:
            most.scatter_add_(-1, want["top_ids"], 4 * U * dtop.double().abs() / temperature)
        at = torch.where(targets != ignore_index, targets, 0)[..., None]
        most.scatter_add_(-1, at, 8 * U * (dlp.double().abs()[..., None] + w[..., None]) / temperature)
        _within(got, want["dlogits"], most, "dlogits")
    return r


VOCABS = [1, 2, 5, 31, 33, 257, 1000, 4099, 8192, 32000, 50257, 131075]


@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes(cuda, V, dtype):
    lead = (3,) if V > 40000 else (2, 7)
    logits = _logits(lead, V, dtype, seed=V)
    targets = torch.randint(0, V, lead, generator=torch.Generator().manual_seed(V + 1))
    targets.view(-1)[1] = -100
    for top_k, temperature in ((min(V, 32), 1.0), (0, 0.7), (min(V, 5), 2.5)):
        _check_token(cuda, logits, targets, top_k, temperature)


@pytest.mark.parametrize("rows", [1, 2, 40, 150, 700])
@pytest.mark.parametrize("V", [4000, 33333])
def test_row_counts(cuda, rows, V):
    """Few rows are split over several blocks; many are not."""
    logits = _logits((rows,), V, torch.bfloat16, seed=rows)
    targets = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(3))
    _check_token(cuda, logits, targets, 9, 1.0, grads=rows < 100)


def test_largest_vocabulary(cuda):
    V = 1 << 20
    logits = _logits((2,), V, torch.float32)
    _check_token(cuda, logits, torch.tensor([V - 1, 0]), 32, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_rows(cuda, dtype):
    """-inf in places, in all but one, in all; the type's lowest value in all
    or in some; one value for all; a target that is masked."""
    V = 5000
    low = torch.finfo(dtype).min
    logits = _logits((12,), V, dtype)
    logits[0, ::2] = -INF
    logits[1, :] = -INF
    logits[1, 4321] = -2.0
    logits[2, :] = -INF
    logits[3, 100:] = low
    logits[4, :] = low
    logits[5, :] = 1.25
    logits[6, 17:] = -INF  # fewer left than alternatives are asked for
    logits[7, :] = torch.finfo(dtype).max
    logits[8, :] = 0.0
    logits[8, 1::2] = -0.0
    logits[9, 3000:] = -INF
    logits[10, :4000] = -INF
    targets = torch.tensor([1, 4321, 7, 4000, 3, 9, 2000, 0, 1, 2999, 3999, -100])
    for temperature in (1.0, 0.5, 3.0):
        _check_token(cuda, logits, targets, 20, temperature)


def test_alternatives_in_adversarial_orders(cuda):
    """Rows where every thread meets larger values later, where a few threads
    hold all of the largest, and where ties fill the row."""
    V = 40000
    j = torch.arange(V)
    rows = torch.stack([
        j / 100.0, -j / 100.0, (j % 8192 < 8).float() * (5 + j / 8192), (j % 256 == 3) * 1.0 + (j % 4096 == 3) * j / 1e5,
        ((j // 16) % 8192 == 0) * 4.0, (j % 7).float(), (j >= V - 40) * 3.0, (j < 33) * 3.0, (j % 4096 < 512) * 1.0 + j * 1e-6,
        torch.where(j % 1024 < 100, 9.0 - (j % 1024) * 1e-3, 0.0)])
    targets = torch.arange(len(rows))
    for dtype in (torch.float32, torch.bfloat16):
        _check_token(cuda, rows.to(dtype), targets, 32, 1.0, grads=False)
        _check_token(cuda, rows.to(dtype), targets, 1, 1.0, grads=False)
        _check_token(cuda, rows[:3].to(dtype).repeat(120, 1), targets[:3].repeat(120), 32, 1.0, grads=False)


def test_strides_and_alignment(cuda):
    """Slices of positions, of a padded vocabulary, off any 16-byte boundary,
    rows given in another order, four dimensions, one dimension."""
    from pulsartecture_b200 import token_logprobs

    base = _logits((3, 9), 1029, torch.bfloat16)
    on = base.to(cuda)
    g = torch.Generator().manual_seed(5)
    for cut in ((slice(None), slice(0, -1), slice(None)), (slice(None), slice(None), slice(0, 1000)),
                (slice(1, None), slice(2, None, 3), slice(3, 1022)), (slice(None), slice(4, 5), slice(1, None))):
        view = base[cut]
        targets = torch.randint(0, view.shape[-1], view.shape[:-1], generator=g)
        _check_token(cuda, view, targets, 3, 1.0, on=on[cut])
    swapped = base.transpose(0, 1)
    targets = torch.randint(0, 1029, (9, 3), generator=g)
    _check_token(cuda, swapped, targets, 3, 1.0, on=on.transpose(0, 1))
    four = base.reshape(3, 3, 3, 1029)[:, :, :2]
    _check_token(cuda, four, torch.randint(0, 1029, (3, 3, 2), generator=g), 3, 1.0, on=on.reshape(3, 3, 3, 1029)[:, :, :2])
    other = base[0].t()  # the vocabulary along the strided dimension
    _check_token(cuda, other, torch.randint(0, 9, (1029,), generator=g), 3, 1.0, on=on[0].t())
    one = token_logprobs(on[0, 0], torch.tensor(5, device=cuda), top_k=2)
    assert one.logprobs.shape == () and one.top_ids.shape == (2,)
    row = on[0, :1].expand(4, 1029)
    _check_token(cuda, base[0, :1].expand(4, 1029), torch.tensor([1, 2, 3, 4]), 2, 1.0, on=row)


def test_ignored_targets(cuda):
    from pulsartecture_b200 import token_logprobs

    logits = _logits((6,), 700, torch.float32)
    targets = torch.tensor([3, 0, 3, 699, 0, 1])
    _check_token(cuda, logits, targets, 4, 1.0, ignore_index=3)
    leaf = logits.to(cuda).requires_grad_()
    r = token_logprobs(leaf, torch.full((6,), -100, device=cuda))
    assert not r.logprobs.any() and (r.entropy > 1).all()
    assert r.top_ids is None and r.top_logprobs is None
    g, = torch.autograd.grad(r.logprobs.sum(), leaf)
    assert not g.any()


def test_rows_without_a_distribution(cuda):
    """A NaN or +inf makes its own row NaN; nothing but -inf makes zeros."""
    from pulsartecture_b200 import token_logprobs

    for rows in (5, 400):
        logits = _logits((rows,), 3001, torch.float32).to(cuda)
        logits[1, 2900] = float("nan")
        logits[2, 3000] = INF
        logits[3] = -INF
        leaf = logits.requires_grad_()
        targets = torch.zeros(rows, dtype=torch.int64, device=cuda)
        r = token_logprobs(leaf, targets, top_k=2)
        g, = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum() + r.top_logprobs.sum(), leaf)
        bad = torch.zeros(rows, dtype=torch.bool, device=cuda)
        bad[1:3] = True
        for t in (r.logprobs, r.entropy, r.top_logprobs[:, 0], g[:, 7]):
            assert torch.equal(torch.isnan(t), bad)
        assert torch.isnan(g[1:3]).all() and (r.top_ids[1:3] == -1).all()
        assert r.logprobs[3] == -INF and r.entropy[3] == 0 and r.top_ids[3].tolist() == [0, 1] and not g[3].any()


def test_bad_targets_are_reported(cuda):
    from pulsartecture_b200 import _lib, token_logprobs
    from pulsartecture_b200.backend.interface import device_status

    device_status()
    logits = _logits((4,), 100, torch.float32).to(cuda).requires_grad_()
    r = token_logprobs(logits, torch.tensor([5, 100, -1, 2 ** 40 + 1], device=cuda))
    g, = torch.autograd.grad(r.logprobs.sum(), logits)
    assert torch.isnan(r.logprobs).tolist() == [False, True, True, True] and torch.isfinite(r.entropy).all()
    assert torch.isnan(g).all(1).tolist() == [False, True, True, True]
    with pytest.raises(_lib.FaklaError) as e:
        device_status()
    assert e.value.status == 1
    device_status()


def test_single_gradients(cuda):
    """Each result alone, and none of them."""
    from pulsartecture_b200 import token_logprobs

    logits, targets = _logits((5,), 900, torch.float32), torch.tensor([1, 2, 3, -100, 5])
    g = torch.Generator().manual_seed(6)
    for which in range(3):
        leaf = logits.to(cuda).requires_grad_()
        r = token_logprobs(leaf, targets.to(cuda), top_k=3)
        given = torch.randn(r[which].shape, generator=g)
        args = [None, None, None]
        args[which] = given
        want = O.token_logprobs(logits, targets, 3, 1.0, -100, *args)["dlogits"]
        got, = torch.autograd.grad(r[which], leaf, given.to(cuda))
        # at most 3 + 1 given values of size |g| meet p and log p of size <= 16
        _within(got, want, torch.full_like(want, 64 * U * float(given.abs().max()) * 4), str(which))
    assert not r.top_ids.requires_grad


def test_gradient_against_differences(cuda):
    from pulsartecture_b200 import distill_topk, token_logprobs

    V = 50
    logits, targets = _logits((3,), V, torch.float32, scale=1.0), torch.tensor([4, 7, 49])
    g = torch.Generator().manual_seed(8)
    d = torch.randn(3, V, generator=g).double()
    ids = torch.stack([torch.randperm(V, generator=g)[:6] for _ in range(3)])
    teacher = torch.randn(3, 6, generator=g)
    lse = torch.logsumexp(teacher, -1) + 0.4
    leaf = logits.to(cuda).requires_grad_()
    r = token_logprobs(leaf, targets.to(cuda), temperature=0.8)
    cases = [(r.logprobs.sum() + r.entropy.sum(),
              lambda z: sum(float(v.sum()) for k, v in O.token_logprobs(z, targets, 0, 0.8).items() if k in ("logprobs", "entropy")))]
    for e in (None, lse):
        loss = distill_topk(leaf, ids.to(cuda), teacher.to(cuda), None if e is None else e.to(cuda), temperature=0.8)
        cases.append((loss.sum(), lambda z, e=e: float(O.distill(z, ids, teacher, e, 0.8)["loss"].sum())))
    for got, f in cases:
        grad, = torch.autograd.grad(got, leaf)
        # central differences in float64: off by eps^2 of the third derivative
        eps = 1e-4
        want = (f(logits.double() + eps * d) - f(logits.double() - eps * d)) / (2 * eps)
        scale = float((grad.cpu().double().abs() * d.abs()).sum())
        assert abs(float((grad.cpu().double() * d).sum()) - want) <= 1e-5 * scale


def _check_distill(cuda, logits, ids, teacher, lse, temperature, on=None, grads=True):
    from pulsartecture_b200 import distill_topk

    V = logits.shape[-1]
    lead = logits.shape[:-1]
    dloss = torch.randn(lead, generator=torch.Generator().manual_seed(9))
    want = O.distill(logits, ids, teacher, lse, temperature, dloss)
    on = logits.to(cuda) if on is None else on
    leaf = on.detach().requires_grad_(grads)
    loss = distill_topk(leaf, ids.to(cuda), teacher.to(cuda), None if lse is None else lse.to(cuda), temperature=temperature)
    assert loss.shape == lead and loss.dtype == torch.float32
    p = want["p"]
    lp = torch.log(p.clamp_min(1e-300))
    err = _sum_error(V, lp, p)
    # the teacher's side: t / temperature - lse is rounded at the size of its
    # terms; what is left over, 1 - sum q, at K units. Each q (log q - log p) is
    # off by q's relative error times (1 + |log q - log p|), and log p by `err`.
    # (an entry at -inf has q = 0, exactly)
    size = torch.where(teacher == -INF, 0.0, teacher.double().abs()).amax(-1) / temperature + (0 if lse is None else lse.double().abs())
    qerr = U * (8 + 4 * size + 2 * ids.shape[-1])
    gap = 1 + lp.abs().amax(-1)
    _within(loss, want["loss"], (qerr * gap + 2 * err + 8 * U * gap) * 2, "loss")
    if grads:
        got, = torch.autograd.grad(loss, leaf, dloss.to(cuda))
        c = dloss.double().abs()[..., None] / temperature
        most = c * p * (2 * err + 2 * qerr + U * (16 + 4 * gap))[..., None]
        if lse is not None:  # p_j q_r / p_r <= q_r, off by the error of q_r, itself at most qerr
            most = most + c * (2 * qerr)[..., None] * torch.ones_like(p)
        at = ids.clamp_min(0)
        most.scatter_add_(-1, at, (c * (2 * qerr)[..., None]).expand(at.shape))
        _within(got, want["dlogits"], most + 4 * U * want["dlogits"].abs(), "dlogits")


def _teacher(lead, V, K, seed, temperature):
    full = torch.randn(*lead, V, generator=torch.Generator().manual_seed(seed)) * 3
    top, ids = torch.topk(full, K, dim=-1)
    return ids, top, torch.logsumexp(full / temperature, -1), full


@pytest.mark.parametrize("V,K", [(1, 1), (5, 5), (33, 7), (1000, 64), (4099, 256), (32000, 50), (50257, 17)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_distill_sizes(cuda, V, K, dtype, temperature):
    lead = (2, 3)
    ids, top, lse, full = _teacher(lead, V, K, V + K, temperature)
    logits = (full * 0.7 + torch.randn(*lead, V, generator=torch.Generator().manual_seed(K))).to(dtype)
    order = torch.randperm(K, generator=torch.Generator().manual_seed(2))  # in no order
    ids, top = ids[..., order], top[..., order]
    _check_distill(cuda, logits, ids, top, None, temperature)
    if K < V:  # with all of the vocabulary kept, what is left over is rounding
        _check_distill(cuda, logits, ids, top, lse, temperature)
    short = torch.where(torch.rand(*lead, K, generator=torch.Generator().manual_seed(4)) < 0.4, -1, ids)
    short[0, 0] = -1  # nothing kept
    _check_distill(cuda, logits, short, top, None, temperature)
    _check_distill(cuda, logits, short, top, lse, temperature)


@pytest.mark.parametrize("rows", [1, 60, 500])
def test_distill_row_counts(cuda, rows):
    V, K = 9000, 20
    ids, top, lse, full = _teacher((rows,), V, K, rows, 1.0)
    logits = (full + 0.5 * torch.randn(rows, V, generator=torch.Generator().manual_seed(1))).bfloat16()
    _check_distill(cuda, logits, ids, top, lse, 1.0)
    _check_distill(cuda, logits, ids, top, None, 1.0)


def test_distill_repeated_ids_and_masks(cuda):
    V, K = 600, 8
    ids, top, lse, full = _teacher((6,), V, K, 3, 1.0)
    logits = full.clone()
    ids[0, 3] = ids[0, 0]  # the same token twice counts twice
    ids[1, :] = ids[1, 0]
    top[2, 2:] = -INF      # entries that the teacher gives nothing
    logits[3, ids[3, 0] + 1 - 2 * (ids[3, 0] == V - 1)] = -INF
    keep = torch.ones(V, dtype=torch.bool)
    keep[ids[4]] = False
    logits[4, keep] = -30.0  # the model puts nearly nothing outside of the entries
    top[5] = -INF
    lse2 = lse + 0.7
    _check_distill(cuda, logits, ids, top, None, 1.0)
    for r in (2, 3, 4, 5):
        _check_distill(cuda, logits[r:r + 1], ids[r:r + 1], top[r:r + 1], lse2[r:r + 1], 1.0)
    q = torch.exp(top[:2].double() - lse2[:2, None].double())
    assert (q.sum(-1) < 1).all()
    _check_distill(cuda, logits[:2], ids[:2], top[:2], lse2[:2], 1.0)


@pytest.mark.parametrize("rows,V", [(3, 2003), (2, 40001), (700, 1000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distill_small_divergences(cuda, rows, V, dtype):
    """Entries that hold little: the rest's class, q_r log(q_r / p_r) with both
    near 1, keeps its digits. Few rows are split over a cluster's blocks; one
    entry is named twice, one lies at a row's unaligned end."""
    from pulsartecture_b200 import distill_topk

    T = 2.0
    g = torch.Generator().manual_seed(V)
    full = torch.randn(rows, V, generator=g)
    logits = (full + 0.5 * torch.randn(rows, V, generator=g)).to(dtype)
    ids = torch.tensor([V // 3, V - 1, V // 3, -1]).expand(rows, 4).contiguous()
    top = full.gather(-1, ids.clamp_min(0))
    lse = torch.logsumexp(full.double() / T, -1).float()
    leaf = logits.to(cuda).requires_grad_()
    dloss = torch.ones(rows)
    want = O.distill(logits, ids, top, lse, T, dloss)
    loss = distill_topk(leaf, ids.to(cuda), top.to(cuda), lse.to(cuda), temperature=T)
    p = want["p"]
    lp = torch.log(p)
    # Q and P are off by their relative errors: the exponentials', 4u, and their
    # arguments' (teacher: terms up to `size`; model: `err` and 4 |log p| u); the
    # rest's class is q_r log1p((P - Q) / p_r), off by those of P and Q and, with
    # q_r and p_r near 1, by 8u of itself, the entries' terms q (log q - log p)
    # by q times both and 8u of themselves
    err = _sum_error(V, lp, p)
    q = torch.exp(top.double() / T - lse.double()[:, None])[:, :3]
    Q, P = q.sum(-1), p[:, [V // 3, V - 1]].sum(-1)
    assert float(Q.max()) < 0.03 and float(P.max()) < 0.03
    size = (top.double().abs() / T).amax(-1) + lse.double().abs()
    most = lp.abs().amax(-1)
    rel_q, rel_p = U * (8 + 4 * size), err + U * (8 + 4 * most)
    terms = (q * (torch.log(q) - lp.gather(-1, ids[:, :3]))).sum(-1).abs()
    tol = 1.1 * (2 * (Q * rel_q + P * rel_p) + Q * (rel_q + rel_p)) + 8 * U * (terms + Q + P)
    _within(loss, want["loss"], tol, "loss")
    # a logit that is no entry: p_j (Q - P) / p_r, p_j's relative error and that of Q - P
    got, = torch.autograd.grad(loss, leaf, dloss.to(cuda))
    rest = torch.ones(V, dtype=torch.bool)
    rest[ids[0, :3]] = False
    off = p * (1.1 * (Q * rel_q + P * rel_p) + 8 * U * (Q + P))[:, None] + (rel_p[:, None] + 8 * U) * want["dlogits"].abs()
    _within(got[:, rest], want["dlogits"][:, rest], off[:, rest] / T, "dlogits")


@pytest.mark.parametrize("V", [259, 4099, 40001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distill_neighbouring_entries(cuda, V, dtype):
    """256 entries side by side, at a row's start, at its end and in between:
    vectors of nothing but entries, and rows that start on no vector."""
    rows, K = 6, 256
    full = torch.randn(rows, V, generator=torch.Generator().manual_seed(V)) * 2
    at = torch.tensor([0, V - K, (V - K) // 2, 0, V - K, (V - K) // 3])
    ids = at[:, None] + torch.arange(K)
    ids[3:] = ids[3:].flip(-1)
    ids[2, 7] = ids[2, 200]
    lse = torch.logsumexp(full, -1)
    logits = (full + 0.5 * torch.randn(rows, V, generator=torch.Generator().manual_seed(1))).to(dtype)
    _check_distill(cuda, logits, ids, full.gather(-1, ids), None, 1.0)
    _check_distill(cuda, logits, ids, full.gather(-1, ids), lse + 0.7, 1.0)


@pytest.mark.parametrize("rows,V", [(3, 40001), (200, 1000)])
@pytest.mark.parametrize("scale", [1.5, 3.0, 8.0, 1e6])
def test_distill_model_sharper_than_the_teacher(cuda, rows, V, scale):
    """The model leaves less than the teacher outside of the entries: a little,
    much (its sum is then taken on its own), nothing."""
    ids, top, lse, full = _teacher((rows,), V, 40, 5, 1.0)
    _check_distill(cuda, full * scale, ids, top, lse, 1.0, grads=scale < 1e6)


def test_distill_largest_vocabulary(cuda):
    """One block to a row of 2^20 fp32 logits in the backward: the most shared memory."""
    from pulsartecture_b200 import distill_topk

    rows, V = 600, 1 << 20
    leaf = torch.zeros(rows, V, device=cuda).requires_grad_()
    ids = torch.tensor([[5, V - 1, V // 2, V // 2]], device=cuda).expand(rows, 4)
    loss = distill_topk(leaf, ids, torch.zeros(rows, 4, device=cuda))
    # q = 1/4 each: log(1/4) - log(1/V); sums of equal powers of two are exact
    _within(loss, torch.tensor(18 * math.log(2.0)).double(), torch.tensor(16 * U * 13), "loss")
    g, = torch.autograd.grad(loss.sum(), leaf)
    want = torch.full((V,), 2.0 ** -20, dtype=torch.float64)
    want[[5, V - 1]] -= 0.25
    want[V // 2] -= 0.5
    for r in (0, 333, rows - 1):
        _within(g[r], want, 16 * U * want.abs(), "dlogits")


def test_distill_rows_without_a_distribution(cuda):
    from pulsartecture_b200 import _lib, distill_topk
    from pulsartecture_b200.backend.interface import device_status

    device_status()
    V, K = 700, 4
    ids, top, lse, full = _teacher((6,), V, K, 3, 1.0)
    logits = full.clone()
    logits[0] = -INF
    logits[1, ids[1, 2]] = -INF  # the teacher gives it something: infinite
    logits[2, 5] = float("nan")
    ids[3, 1], ids[4, 2] = V, -2
    for e in (None, lse):
        leaf = logits.to(cuda).requires_grad_()
        loss = distill_topk(leaf, ids.to(cuda), top.to(cuda), None if e is None else e.to(cuda))
        g, = torch.autograd.grad(loss.sum(), leaf)
        assert loss[0] == INF and not g[0].any()
        assert loss[1] == INF and torch.isfinite(g[1]).all()
        assert torch.isnan(loss).tolist() == [False, False, True, True, True, False]
        assert torch.isnan(g[2:5]).all() and torch.isfinite(g[5]).all()
        with pytest.raises(_lib.FaklaError):
            device_status()


def test_distill_strides_and_types(cuda):
    from pulsartecture_b200 import distill_topk

    base = _logits((3, 9), 1029, torch.bfloat16)
    on = base.to(cuda)
    for cut in ((slice(None), slice(0, -1), slice(None)), (slice(1, None), slice(2, None, 3), slice(3, 1022))):
        ids, top, lse, _ = _teacher(base[cut].shape[:-1], base[cut].shape[-1], 10, 3, 1.0)
        _check_distill(cuda, base[cut], ids, top, lse, 1.0, on=on[cut])
    ids, top, lse, _ = _teacher((3, 9), 1029, 10, 3, 1.0)
    a = distill_topk(on, ids.to(cuda), top.bfloat16().to(cuda), lse.double().to(cuda))
    b = distill_topk(on, ids.to(cuda), top.bfloat16().float().to(cuda), lse.to(cuda))
    assert torch.equal(a, b)


def test_rows_past_32_bits(cuda):
    """More than 2^31 logits: the last rows are read and written in their places."""
    from pulsartecture_b200 import distill_topk, token_logprobs

    V = 32000
    rows = 2 ** 31 // V + 40
    logits = torch.zeros(rows, V, device=cuda, dtype=torch.bfloat16)
    tail = _logits((8,), V, torch.bfloat16)
    logits[-8:] = tail.to(cuda)
    leaf = logits.requires_grad_()
    targets = torch.full((rows,), 11, device=cuda)
    r = token_logprobs(leaf, targets, top_k=2)
    want = O.token_logprobs(tail, torch.full((8,), 11), 2, 1.0, -100, torch.ones(8))
    _within(r.logprobs[-8:], want["logprobs"], _sum_error(V, want["lp"], want["p"]) + 60 * U, "logprobs")
    assert torch.equal(r.top_ids[-8:].cpu(), want["top_ids"]) and r.top_ids[0].tolist() == [0, 1]
    g, = torch.autograd.grad(r.logprobs.sum(), leaf)
    _within(g[-8:], want["dlogits"], 400 * U * want["p"] + 16 * U, "dlogits")
    del g
    ids = targets[:, None]
    loss = distill_topk(leaf, ids, torch.zeros(rows, 1, device=cuda))
    # one entry: q = 1, the loss is the token's -log p
    _within(loss[-8:], -want["logprobs"], _sum_error(V, want["lp"], want["p"]) + 60 * U, "loss")
    g, = torch.autograd.grad(loss.sum(), leaf)
    _within(g[-8:], -want["dlogits"], 400 * U * want["p"] + 16 * U, "dlogits")


def test_captured_and_on_another_stream(cuda):
    """Forward and backward captured and replayed on new inputs equal eager
    calls bit for bit; so do calls on a side stream. Rows are split over blocks
    in one case and not in the other."""
    from pulsartecture_b200 import distill_topk, token_logprobs

    for rows, V in ((3, 20000), (900, 1111), (600, 140000)):
        def inputs(seed):
            ids, top, lse, full = _teacher((rows,), V, 12, seed, 1.0)
            return [t.to(cuda) for t in (full.bfloat16(), ids[:, 3].contiguous(), ids, top, lse)]

        def work(logits, targets, ids, top, lse):
            leaf = logits.detach().requires_grad_()
            r = token_logprobs(leaf, targets, top_k=6)
            loss = distill_topk(leaf, ids, top, lse)
            g1, = torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], leaf,
                                      [torch.ones_like(r.logprobs), torch.ones_like(r.entropy), torch.ones_like(r.top_logprobs)])
            g2, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
            return [t.detach() for t in (*r, loss, g1, g2)]

        held_in = inputs(1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            early = work(*held_in)
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(early, work(*held_in)):
            assert torch.equal(a, b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = work(*held_in)
        for seed in (2, 3):
            new = inputs(seed)
            for a, b in zip(held_in, new):
                a.copy_(b)
            graph.replay()
            for a, b in zip(held, work(*new)):
                assert torch.equal(a, b)


def test_no_rows(cuda):
    from pulsartecture_b200 import distill_topk, token_logprobs

    logits = torch.empty(2, 0, 50, device=cuda, requires_grad=True)
    r = token_logprobs(logits, torch.empty(2, 0, dtype=torch.int64, device=cuda), top_k=3)
    assert r.logprobs.shape == (2, 0) and r.entropy.shape == (2, 0) and r.top_ids.shape == (2, 0, 3)
    (r.logprobs.sum() + r.entropy.sum()).backward()
    loss = distill_topk(logits, torch.empty(2, 0, 4, dtype=torch.int64, device=cuda), torch.empty(2, 0, 4, device=cuda))
    assert loss.shape == (2, 0)
    loss.sum().backward()


def test_gradient_of_no_alternatives(cuda):
    from pulsartecture_b200 import token_logprobs

    logits = torch.empty(0, 50, device=cuda, requires_grad=True)
    r = token_logprobs(logits, torch.empty(0, dtype=torch.int64, device=cuda), top_k=3)
    assert r.top_logprobs.shape == (0, 3)
    r.top_logprobs.sum().backward()
    assert logits.grad.shape == (0, 50)


def test_refusals_on_device_tensors(cuda):
    from pulsartecture_b200 import distill_topk, token_logprobs

    z = torch.randn(3, 40, device=cuda)
    t = torch.zeros(3, dtype=torch.int64, device=cuda)
    ids = torch.zeros(3, 4, dtype=torch.int64, device=cuda)
    top = torch.zeros(3, 4, device=cuda)
    for call in (lambda: token_logprobs(z, t.int()), lambda: token_logprobs(z, t[:2]), lambda: token_logprobs(z, t, top_k=41),
                 lambda: token_logprobs(z, t, top_k=33), lambda: token_logprobs(z, t, top_k=-1), lambda: token_logprobs(z.half(), t),
                 lambda: token_logprobs(z, t, temperature=0.0), lambda: token_logprobs(z, t, temperature=float("nan")),
                 lambda: token_logprobs(z, t.cpu()), lambda: token_logprobs(z[:, :0], t),
                 lambda: distill_topk(z, ids.int(), top), lambda: distill_topk(z, ids, top[:, :3]),
                 lambda: distill_topk(z, ids[:, :0], top[:, :0]), lambda: distill_topk(z, ids, top, t.float()[:2]),
                 lambda: distill_topk(z, ids, top, temperature=-1.0), lambda: distill_topk(z, ids, top.cpu()),
                 lambda: distill_topk(z, ids.repeat(1, 65), top.repeat(1, 65)), lambda: distill_topk(z, ids, ids)):
        with pytest.raises(RuntimeError):
            call()
    leaf = z.clone().requires_grad_()
    first, = torch.autograd.grad(token_logprobs(leaf, t).logprobs.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative, and no silent zero
        first.sum().backward()
