"""The recurrence's and the logits operators' refusals, at the C ABI and in the
torch front end, and the language model's choice of recurrent layers. CPU
only: every call here is refused before a device is touched."""
import ctypes

import pytest
import torch

from pulsartecture_b200 import _lib, distill_topk, gated_scan, gated_scan_step, token_logprobs


def _no_gpu():
    if torch.cuda.is_available():
        pytest.skip("dummy pointers are passed only where no GPU exists")


P = ctypes.c_void_p(16)  # never dereferenced


def test_gated_scan_arguments():
    _no_gpu()
    L = _lib.lib()

    def scan(x=P, gate=P, out=P, B=1, T=1, D=8, act=5, dtype=1):
        return L.fakla_gated_scan(x, gate, out, None, None, None, B, T, D, D, D, D, D, act, 1, dtype, None)

    assert scan(dtype=7) == 1 and b"dtype" in L.fakla_last_error()
    for bad in (dict(x=None), dict(gate=None), dict(out=None), dict(B=0), dict(T=0), dict(D=-1)):
        assert scan(**bad) == 1, bad
    assert scan(act=1) == 2 and b"sigmoid" in L.fakla_last_error()
    assert scan(B=2 ** 40) == 2 and scan(D=2 ** 40) == 2 and scan(B=2 ** 20, D=2 ** 20) == 2
    assert scan() in (4, 7)

    def back(saved=P, dx=P, D=8):
        return L.fakla_gated_scan_backward(P, P, saved, P, None, dx, P, None, 1, 1, D, D, D, D, D, 5, 1, 1, None)

    assert back(saved=None) == 1 and back(dx=None) == 1 and back(D=0) == 1 and back() in (4, 7)
    assert L.fakla_gated_scan_step(P, P, P, None, P, 1, 8, 8, 8, 5, 1, 1, None) == 1
    assert L.fakla_gated_scan_step(P, P, P, P, None, 1, 8, 8, 8, 5, 1, 1, None) == 1
    odd = ctypes.c_void_p(17)
    for bad in (dict(x=odd), dict(gate=odd), dict(out=odd)):
        assert scan(**bad) == 3, bad
    assert back(saved=odd) == 3 and back(dx=odd) == 3
    assert L.fakla_gated_scan_step(P, P, P, P, odd, 1, 8, 8, 8, 5, 1, 1, None) == 3
    assert L.fakla_gated_scan_saved_bytes(2, 129, 10) >= 2 * 10 * 4
    assert L.fakla_gated_scan_saved_bytes(0, 129, 10) == 0


def test_logits_arguments():
    _no_gpu()
    L = _lib.lib()

    def score(logits=P, targets=P, lp=P, top=P, batch=1, rows=1, V=100, k=4, temperature=1.0, dtype=0):
        return L.fakla_token_logprobs(logits, targets, lp, P, top, P, None, batch, rows, V, V, V, k, temperature, -100,
                                      dtype, None)

    for bad in (dict(logits=None), dict(targets=None), dict(lp=None), dict(top=None), dict(batch=0), dict(rows=0),
                dict(V=0), dict(k=-1), dict(k=33), dict(V=3), dict(temperature=0.0), dict(temperature=float("nan")),
                dict(temperature=float("inf")), dict(temperature=-1.0), dict(dtype=2)):
        assert score(**bad) == 1, bad
    assert score(logits=ctypes.c_void_p(18)) == 3  # fp32 from an address off 4 bytes
    assert score(V=2 ** 20 + 1) == 2 and score(rows=2 ** 40) == 2 and score(batch=2 ** 20, rows=2 ** 20) == 2
    assert score() in (4, 7) and score(k=0, top=None) in (4, 7)

    def back(stats=P, ids=P, dtop=None, k=0):
        return L.fakla_token_logprobs_backward(P, P, stats, P, ids, P, P, dtop, P, 1, 1, 100, 100, 100, k, 1.0, -100, 0, None)

    assert back(stats=None) == 1 and back(ids=None, dtop=P, k=2) == 1 and back(dtop=P, k=0) == 1 and back() in (4, 7)

    def distill(ids=P, loss=P, K=4, V=100):
        return L.fakla_distill_topk(P, ids, P, None, loss, None, 1, 1, V, V, V, K, 1.0, 0, None)

    assert distill(ids=None) == 1 and distill(loss=None) == 1 and distill(K=0) == 1 and distill(K=257) == 1
    assert distill(V=2 ** 20 + 1) == 2 and distill() in (4, 7)
    assert L.fakla_distill_topk_backward(P, P, P, None, None, P, P, 1, 1, 100, 100, 100, 4, 1.0, 0, None) == 1


def test_front_end_checks_shapes_types_and_device():
    x, s = torch.zeros(2, 3, 4), torch.zeros(2, 4)
    for call, word in ((lambda: gated_scan(x, x), "CUDA"), (lambda: gated_scan(x[0], x[0]), "B, T, D"),
                       (lambda: gated_scan(x, x[:, :2]), "match"), (lambda: gated_scan(x, x.bfloat16()), "dtype"),
                       (lambda: gated_scan(x, x, gate_act="tanh"), "gate_act"),
                       (lambda: gated_scan_step(x, x, s), "N, D"), (lambda: gated_scan_step(x[:, 0], x[:, 0], s), "CUDA")):
        with pytest.raises(RuntimeError, match=word):
            call()
    z, t = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64)
    for call, word in ((lambda: token_logprobs(z, t), "CUDA"), (lambda: token_logprobs(z, t, temperature=0), "temperature"),
                       (lambda: distill_topk(z, t[:, None], z[:, :1]), "CUDA"),
                       (lambda: distill_topk(z, t[:, None], z[:, :1], temperature=-2), "temperature")):
        with pytest.raises(RuntimeError, match=word):
            call()


def test_recurrent_layers_of_the_model():
    from pulsartecture_b200.attention import GatedRecurrence, TMLinKernelAttn
    from pulsartecture_b200.lm_harness import FaklaLM

    small = dict(vocab=20, d_model=64, n_heads=1, head_dim=64, d_ff=32, n_experts=2, top_k=1)
    m = FaklaLM(n_layers=3, recurrent_layers=(0, 2), **small)
    assert [type(b.attn) for b in m.blocks] == [GatedRecurrence, TMLinKernelAttn, GatedRecurrence]
    for bad in ((3,), (-1,)):
        with pytest.raises(ValueError):
            FaklaLM(n_layers=3, recurrent_layers=bad, **small)
    torch.manual_seed(0)
    a = FaklaLM(n_layers=2, **small)
    torch.manual_seed(0)
    b = FaklaLM(n_layers=2, recurrent_layers=(), **small)
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    with pytest.raises(ValueError):
        GatedRecurrence(8, 0)
    g = GatedRecurrence(8, 4, gate_bias=3.0)
    assert g.init_state(5).shape == (5, 4) and (g.proj.linear.bias[4:] > 2).all()


def test_oracles_agree_with_autograd():
    """The written-out gradients of the oracles against automatic ones."""
    from oracle import logits_oracle, recurrence_oracle

    g = torch.Generator().manual_seed(0)
    x, gate = (torch.randn(2, 9, 3, generator=g, dtype=torch.float64).requires_grad_() for _ in range(2))
    s = torch.randn(2, 3, generator=g, dtype=torch.float64).requires_grad_()
    for act, mix in (("sigmoid", True), ("identity", False), ("identity", True)):
        a = torch.sigmoid(gate) if act == "sigmoid" else gate
        h, hs = s, []
        for t in range(9):
            h = a[:, t] * h + ((1 - a[:, t]) * x[:, t] if mix else x[:, t])
            hs.append(h)
        w = torch.randn(2, 9, 3, generator=g, dtype=torch.float64)
        want = torch.autograd.grad((torch.stack(hs, 1) * w).sum() + h.sum(), [x, gate, s])
        val, _ = recurrence_oracle.scan(x.detach(), gate.detach(), s.detach(), act, mix, dout=w, dstate=torch.ones(2, 3))
        for n, v in zip(["dx", "dgate", "dstate"], want):
            assert torch.allclose(val[n], v, rtol=1e-12, atol=1e-12)
    z = torch.randn(4, 11, generator=g, dtype=torch.float64).requires_grad_()
    lp = torch.log_softmax(z / 0.7, -1)
    p = lp.exp()
    t = torch.tensor([3, -100, 0, 10])
    dlp, dent, dtop = (torch.randn(*sh, generator=g, dtype=torch.float64) for sh in ((4,), (4,), (4, 3)))
    top = torch.topk(lp, 3).values
    pick = torch.where(t >= 0, lp.gather(-1, t.clamp_min(0)[:, None])[:, 0], 0.0)
    want, = torch.autograd.grad((pick * dlp).sum() - ((p * lp).sum(-1) * dent).sum() + (top * dtop).sum(), z, retain_graph=True)
    got = logits_oracle.token_logprobs(z.detach(), t, 3, 0.7, -100, dlp, dent, dtop)
    assert torch.allclose(got["dlogits"], want, rtol=1e-12, atol=1e-12)
    ids = torch.tensor([[1, 2, 3], [4, -1, 5], [-1, -1, -1], [0, 9, 10]])
    teacher = torch.randn(4, 3, generator=g, dtype=torch.float64)
    for lse in (None, torch.logsumexp(teacher / 0.7, -1) + 0.3):
        total = 0
        for r in range(4):
            i = ids[r][ids[r] >= 0]
            tr = teacher[r][ids[r] >= 0] / 0.7
            if len(i):
                q = torch.softmax(tr, 0) if lse is None else torch.exp(tr - lse[r])
                total = total + (q * (q.log() - lp[r][i])).sum() * dlp[r]
                if lse is not None:
                    qr, pr = 1 - q.sum(), 1 - p[r][i].sum()
                    total = total + qr * (qr.log() - pr.log()) * dlp[r]
        want, = torch.autograd.grad(total, z, retain_graph=True)
        got = logits_oracle.distill(z.detach(), ids, teacher, lse, 0.7, dlp)
        assert torch.allclose(got["dlogits"], want, rtol=1e-10, atol=1e-10)


def test_logits_pointers_off_their_elements():
    """Every pointer of the logits entry points is refused where it is not on a
    multiple of its element: a kernel could not read or write there."""
    _no_gpu()
    L = _lib.lib()
    calls = {
        # pointers, in order: T = logits' type (fp32 here), f = fp32, i = int64
        "fakla_token_logprobs": ("Tifffif", [1, 1, 100, 100, 100, 4, 1.0, -100, 0]),
        "fakla_token_logprobs_backward": ("TiffifffT", [1, 1, 100, 100, 100, 4, 1.0, -100, 0]),
        "fakla_distill_topk": ("Tiffff", [1, 1, 100, 100, 100, 4, 1.0, 0]),
        "fakla_distill_topk_backward": ("TiffffT", [1, 1, 100, 100, 100, 4, 1.0, 0]),
    }
    for name, (kinds, rest) in calls.items():
        fn = getattr(L, name)
        assert fn(*[P] * len(kinds), *rest, None) in (4, 7), name
        for n, kind in enumerate(kinds):
            for off in (18, 20):
                args = [P] * len(kinds)
                args[n] = ctypes.c_void_p(off)
                assert (fn(*args, *rest, None) == 3) == (off % (8 if kind == "i" else 4) != 0), (name, n, off)


def test_states_that_overlap_in_part():
    """state_out is state_in or apart from it: blocks read the one while others
    write the other."""
    _no_gpu()
    L = _lib.lib()
    N, D = 4, 8
    size = N * D * 4
    for off, refused in ((0, False), (4, True), (size - 4, True), (-4, True), (4 - size, True), (size, False), (-size, False)):
        a, b = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + off)
        for rc in (L.fakla_gated_scan_step(P, P, P, a, b, N, D, D, D, 5, 1, 1, None),
                   L.fakla_gated_scan(P, P, P, a, b, None, N, 3, D, 3 * D, D, 3 * D, D, 5, 1, 1, None)):
            assert (rc == 1 and b"overlap" in L.fakla_last_error()) if refused else rc in (4, 7), off
