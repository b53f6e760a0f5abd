"""gated_scan and gated_scan_step against the float64 recurrence.

Bounds are derived, element by element (oracle/recurrence_oracle.py): every
factor off by at most k units of 2^-24. An exponential of |g| <= 16 on the fast
path is off by 2 + 1.2 |g| < 22 ulp, so by 44 units, the reciprocal by 4, the
remaining products and sums by a handful: k = 64. float32 gates take the
accurate exponential, 2 ulp: k = 16. Storing bf16 adds half a step, 2^-8 of the
value (GPU only).
"""
import pytest
import torch

from oracle import recurrence_oracle as O

pytestmark = pytest.mark.gpu

FACTOR = {torch.float32: 16.0, torch.bfloat16: 64.0}


def _inputs(B, T, D, dtype, act, seed=0, state=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T, D, generator=g).to(dtype)
    gate = (torch.randn(B, T, D, generator=g) * 2 + 2).clamp(-16, 16)
    gate = (gate if act == "sigmoid" else torch.sigmoid(gate) * torch.where(torch.rand(B, T, D, generator=g) < 0.2, -1, 1)).to(dtype)
    s = torch.randn(B, D, generator=g) if state else None
    return x, gate, s


def _close(got, value, bound, name):
    got = got.detach().cpu()
    step = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    # the stored value is a rounding of something within `bound` of `value`
    # (the smallest numbers round to multiples of 2^-133 in bf16, 2^-149 in fp32)
    tol = bound + step * (value.abs() + bound) + O.U * value.abs() + 2.0 ** -133
    off = (got.double() - value).abs()
    assert torch.isfinite(got).all(), name
    assert bool((off <= tol).all()), (name, float((off / tol).max()))


SIZES = [(1, 1, 1), (2, 1, 7), (1, 2, 64), (3, 5, 33), (1, 127, 8), (2, 128, 65), (2, 129, 130), (1, 1000, 515),
         (5, 257, 64), (1, 4100, 40), (40, 17, 192),
         # batches that put one, two and four blocks on a sequence
         (300, 390, 33), (150, 520, 64), (75, 1100, 64), (2, 2111, 64), (10, 1030, 256)]


@pytest.mark.parametrize("B,T,D", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act,mix", [("sigmoid", True), ("sigmoid", False), ("identity", True), ("identity", False)])
def test_scan_and_gradients(cuda, B, T, D, dtype, act, mix):
    from pulsartecture_b200 import gated_scan

    state = (B + T) % 2 == 0
    x, gate, s = _inputs(B, T, D, dtype, act, state=state)
    g = torch.Generator().manual_seed(1)
    dout, dstate = torch.randn(B, T, D, generator=g).to(dtype), torch.randn(B, D, generator=g)
    val, bound = O.scan(x, gate, s, act, mix, FACTOR[dtype], dout, dstate)
    with torch.no_grad():
        plain, end = gated_scan(x.to(cuda), gate.to(cuda), None if s is None else s.to(cuda), gate_act=act, mix=mix)
    leaves = [t.to(cuda).requires_grad_() for t in (x, gate, s) if t is not None]
    out, final = gated_scan(leaves[0], leaves[1], leaves[2] if state else None, gate_act=act, mix=mix)
    assert torch.equal(out, plain) and torch.equal(final, end)
    grads = torch.autograd.grad([out, final], leaves, [dout.to(cuda), dstate.to(cuda)])
    _close(out, val["out"], bound["out"], "out")
    _close(final, val["state"], bound["state"], "state")
    for n, got in zip(["dx", "dgate", "dstate"], grads):
        _close(got, val[n], bound[n], n)


def test_gradients_against_differences(cuda):
    from pulsartecture_b200 import gated_scan

    x, gate, s = _inputs(2, 37, 5, torch.float32, "sigmoid")
    leaves = [t.to(cuda).requires_grad_() for t in (x, gate, s)]
    g = torch.Generator().manual_seed(2)
    w = torch.randn(2, 37, 5, generator=g)
    out, final = gated_scan(*leaves)
    grads = torch.autograd.grad([out, final], leaves, [w.to(cuda), torch.ones_like(final)])

    def loss(v):
        o, _ = O.scan(*v)
        return float((o["out"] * w.double()).sum() + o["state"].sum())

    # central differences in float64 along a random direction: off by eps^2 of
    # the third derivative, far below the float32 gradients' own error
    for i, name in enumerate(["x", "gate", "state"]):
        d = torch.randn(leaves[i].shape, generator=g).double()
        eps = 1e-4
        v = [t.double() for t in (x, gate, s)]
        up, down = list(v), list(v)
        up[i], down[i] = v[i] + eps * d, v[i] - eps * d
        want = (loss(up) - loss(down)) / (2 * eps)
        got = float((grads[i].cpu().double() * d).sum())
        scale = float((grads[i].cpu().double().abs() * d.abs()).sum())
        assert abs(got - want) <= 1e-5 * scale, name


def test_only_one_result_has_a_gradient(cuda):
    from pulsartecture_b200 import gated_scan

    x, gate, s = _inputs(2, 150, 66, torch.float32, "sigmoid")
    zero = torch.zeros(2, 66)
    for which in (0, 1):
        leaves = [t.to(cuda).requires_grad_() for t in (x, gate, s)]
        r = gated_scan(*leaves)
        g = torch.Generator().manual_seed(3)
        given = torch.randn(r[which].shape, generator=g)
        grads = torch.autograd.grad(r[which], leaves, given.to(cuda))
        dout, dstate = (given, zero) if which == 0 else (torch.zeros(2, 150, 66), given)
        val, bound = O.scan(x, gate, s, "sigmoid", True, FACTOR[torch.float32], dout, dstate)
        for n, got in zip(["dx", "dgate", "dstate"], grads):
            _close(got, val[n], bound[n], n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,lead", [(64, 0), (64, 1), (65, 0), (8, 3)])
def test_column_blocks_and_expanded_rows(cuda, dtype, D, lead):
    """Both inputs as column blocks of one projection, off its first column;
    a gate shared by the batch; a value shared by all tokens."""
    from pulsartecture_b200 import gated_scan

    B, T = 3, 140
    g = torch.Generator().manual_seed(4)
    both = (torch.randn(B, T, lead + 2 * D, generator=g) + 1).to(dtype)
    x, gate = both[..., lead:lead + D], both[..., lead + D:]
    shared = torch.randn(1, T, D, generator=g).to(dtype).expand(B, T, D)
    still = torch.randn(B, 1, D, generator=g).to(dtype).expand(B, T, D)
    for xs, gs in ((x, gate), (x, shared), (still, gate)):
        dout = torch.randn(B, T, D, generator=g).to(dtype)
        val, bound = O.scan(xs, gs, None, "sigmoid", True, FACTOR[dtype], dout)
        on = both.to(cuda)
        xc = on[..., lead:lead + D] if xs is x else xs[:, :1].to(cuda).expand(B, T, D)
        gc = on[..., lead + D:] if gs is gate else gs[:1].to(cuda).expand(B, T, D)
        xc, gc = xc.detach().requires_grad_(), gc.detach().requires_grad_()
        out, _ = gated_scan(xc, gc)
        dx, dgate = torch.autograd.grad(out, [xc, gc], dout.to(cuda))
        _close(out, val["out"], bound["out"], "out")
        _close(dx, val["dx"], bound["dx"], "dx")
        _close(dgate, val["dgate"], bound["dgate"], "dgate")


def test_gradient_of_a_broadcast_gate_is_its_sum(cuda):
    from pulsartecture_b200 import gated_scan

    x, gate, _ = _inputs(4, 30, 12, torch.float32, "sigmoid", state=False)
    one = gate[:1].to(cuda).requires_grad_()
    out, _ = gated_scan(x.to(cuda), one.expand(4, 30, 12))
    out.sum().backward()
    val, bound = O.scan(x, gate[:1].expand(4, 30, 12), None, "sigmoid", True, 16.0, torch.ones(4, 30, 12))
    _close(one.grad, val["dgate"].sum(0, keepdim=True), bound["dgate"].sum(0, keepdim=True) + 4 * O.U * val["dgate"].abs().sum(0, keepdim=True), "dgate")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_handing_the_state_over_equals_one_call(cuda, dtype):
    from pulsartecture_b200 import gated_scan, gated_scan_step

    B, T, D = 2, 300, 72
    x, gate, s = _inputs(B, T, D, dtype, "sigmoid")
    val, bound = O.scan(x, gate, s, "sigmoid", True, FACTOR[dtype])
    xc, gc, sc = x.to(cuda), gate.to(cuda), s.to(cuda)
    kept = sc.clone()
    parts, state = [], sc
    for t0, t1 in ((0, 1), (1, 130), (130, 256), (256, 290)):
        out, state = gated_scan(xc[:, t0:t1], gc[:, t0:t1], state)
        parts.append(out)
    assert torch.equal(sc, kept)  # the given state is not modified
    for t in range(290, T):
        if t % 2:
            out, same = gated_scan_step(xc[:, t], gc[:, t], state)
            assert same is state
        else:
            new = torch.empty_like(state)
            old = state.clone()
            out, got = gated_scan_step(xc[:, t], gc[:, t], state, new_state=new)
            assert got is new and torch.equal(state, old)
            state = new
        parts.append(out[:, None])
    _close(torch.cat(parts, 1), val["out"], bound["out"], "out")
    _close(state, val["state"], bound["state"], "state")


@pytest.mark.parametrize("N,D", [(1, 1), (3, 7), (2, 64), (300, 130), (70000, 8)])
@pytest.mark.parametrize("act,mix", [("sigmoid", True), ("identity", False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step(cuda, N, D, act, mix, dtype):
    from pulsartecture_b200 import gated_scan_step

    x, gate, s = _inputs(N, 1, D, dtype, act)
    val, bound = O.scan(x, gate, s, act, mix, FACTOR[dtype])
    state = s.to(cuda)
    both = torch.cat([x[:, 0], gate[:, 0]], 1).to(cuda)
    out, _ = gated_scan_step(both[:, :D], both[:, D:], state, gate_act=act, mix=mix)
    _close(out, val["out"][:, 0], bound["out"][:, 0], "out")
    _close(state, val["state"], bound["state"], "state")


def test_gates_at_their_ends(cuda):
    """-inf forgets, +inf keeps; 0 forgets and 1 keeps without a sigmoid."""
    from pulsartecture_b200 import gated_scan

    T, D = 200, 3
    x = torch.randn(1, T, D, generator=torch.Generator().manual_seed(5)).to(cuda)
    s = torch.full((1, D), 7.0, device=cuda)
    keep = torch.full((1, T, D), float("inf"), device=cuda)
    out, end = gated_scan(x, keep, s)
    assert torch.equal(out, s[:, None].expand(1, T, D)) and torch.equal(end, s)
    gate = torch.zeros(1, T, D, device=cuda)
    gate[:, 100] = -float("inf")  # a second document
    leaves = [x.clone().requires_grad_(), gate.clone().requires_grad_()]
    both, _ = gated_scan(*leaves, s)
    second, _ = gated_scan(x[:, 100:], gate[:, 100:])
    assert torch.equal(both[:, 100], x[:, 100])
    assert torch.allclose(both[:, 100:], second, rtol=1e-6, atol=1e-6)
    dx, dgate = torch.autograd.grad(both[:, 100:].sum(), leaves)
    assert not dx[:, :100].any() and not dgate[:, :101].any() and torch.isfinite(dgate).all()
    ones = torch.ones(1, T, D, device=cuda)
    out, _ = gated_scan(torch.ones(1, T, D, device=cuda), ones, gate_act="identity", mix=False)
    assert torch.equal(out[0, :, 0].cpu(), torch.arange(1.0, T + 1))  # a running sum


def test_growing_coefficients_and_non_finite_values_stay_in_their_place(cuda):
    from pulsartecture_b200 import gated_scan

    T, D = 400, 34
    a = torch.full((1, T, D), 1.5, device=cuda)
    x = torch.zeros(1, T, D, device=cuda)
    out, end = gated_scan(x, a, gate_act="identity", mix=False)  # 1.5^400 is past float32, 0 times it is not
    assert not out.any() and not end.any()
    x, gate, _ = _inputs(1, T, D, torch.float32, "sigmoid", state=False)
    val, bound = O.scan(x, gate, None)
    x[0, 250, 3] = float("nan")
    out, end = gated_scan(x.to(cuda), gate.to(cuda))
    hit = torch.zeros(1, T, D, dtype=torch.bool)
    hit[0, 250:, 3] = True
    assert torch.equal(torch.isnan(out).cpu(), hit) and torch.isnan(end[0]).nonzero().flatten().tolist() == [3]
    _close(torch.where(hit.to(cuda), 0.0, out), torch.where(hit, 0.0, val["out"]), bound["out"], "out")


def test_no_tokens(cuda):
    from pulsartecture_b200 import gated_scan, gated_scan_step

    x = torch.empty(2, 0, 5, device=cuda)
    s = torch.randn(2, 5, device=cuda)
    out, end = gated_scan(x, x, s)
    assert out.shape == (2, 0, 5) and torch.equal(end, s) and end.data_ptr() != s.data_ptr()
    out, end = gated_scan(x, x)
    assert torch.equal(end, torch.zeros(2, 5, device=cuda))
    out, end = gated_scan(x[:0], x[:0])
    assert out.shape == (0, 0, 5) and end.shape == (0, 5)
    out, end = gated_scan_step(x[:0, 0:0].reshape(0, 5), x[:0].reshape(0, 5), s[:0])
    assert out.shape == (0, 5)


@pytest.mark.parametrize("shape", [(2, 0, 5), (0, 3, 5), (2, 3, 0)])
def test_gradients_of_nothing(cuda, shape):
    from pulsartecture_b200 import gated_scan

    x, gate = torch.empty(shape, device=cuda, requires_grad=True), torch.empty(shape, device=cuda, requires_grad=True)
    s = torch.randn(shape[0], shape[2], device=cuda, requires_grad=True)
    out, end = gated_scan(x, gate, s)
    assert out.shape == shape and out.is_contiguous()
    (out.sum() + end.sum()).backward()
    assert x.grad.shape == shape and gate.grad.shape == shape and torch.equal(s.grad, torch.ones_like(s))


def test_offsets_past_32_bits(cuda):
    """A batch stride of more than 2^31 elements."""
    from pulsartecture_b200 import gated_scan

    T, D, far = 130, 64, 2 ** 31 + 64
    flat = torch.empty(far + T * 2 * D, device=cuda, dtype=torch.bfloat16)
    x, gate, _ = _inputs(2, T, D, torch.bfloat16, "sigmoid", state=False)
    xs = flat.as_strided((2, T, D), (far, 2 * D, 1))
    gs = flat.as_strided((2, T, D), (far, 2 * D, 1), D)
    xs.copy_(x.to(cuda))
    gs.copy_(gate.to(cuda))
    val, bound = O.scan(x, gate, None, k=64.0, dout=torch.ones(2, T, D))
    xs.requires_grad_()
    out, end = gated_scan(xs, gs)
    _close(out, val["out"], bound["out"], "out")
    dx, = torch.autograd.grad(out, xs, torch.ones_like(out))
    _close(dx, val["dx"], bound["dx"], "dx")


def test_captured_and_on_another_stream(cuda):
    """Forward and backward captured into a graph and replayed on new inputs
    give what eager calls give, bit for bit; so do calls on a side stream."""
    from pulsartecture_b200 import gated_scan, gated_scan_step

    B, T, D = 2, 1500, 96
    x, gate, s = (t.to(cuda) for t in _inputs(B, T, D, torch.bfloat16, "sigmoid"))
    dout = torch.ones(B, T, D, device=cuda, dtype=torch.bfloat16)

    def work(xx, gg, ss):
        xx, gg = xx.detach().requires_grad_(), gg.detach().requires_grad_()
        out, end = gated_scan(xx, gg, ss)
        with torch.no_grad():
            step, last = gated_scan_step(xx[:, 0], gg[:, 0], end.detach(), new_state=torch.empty_like(end))
        return (out.detach(), end.detach(), step, last, *torch.autograd.grad(out, [xx, gg], dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        early = work(x, gate, s)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(early, work(x, gate, s)):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work(x, gate, s)
    for seed in (7, 8):
        nx, ng, ns = (t.to(cuda) for t in _inputs(B, T, D, torch.bfloat16, "sigmoid", seed))
        for old, new in ((x, nx), (gate, ng), (s, ns)):
            old.copy_(new)
        graph.replay()
        for a, b in zip(held, work(nx, ng, ns)):
            assert torch.equal(a, b)


def test_refusals_on_device_tensors(cuda):
    from pulsartecture_b200 import gated_scan, gated_scan_step

    x = torch.randn(2, 4, 6, device=cuda)
    s = torch.zeros(2, 6, device=cuda)
    for call in (lambda: gated_scan(x, x, s.double()), lambda: gated_scan(x, x, s[:, :5]),
                 lambda: gated_scan(x, x, s.cpu()), lambda: gated_scan(x.half(), x.half()),
                 lambda: gated_scan(x, x.cpu()), lambda: gated_scan_step(x[:, 0], x[:, 0], None),
                 lambda: gated_scan_step(x[:, 0], x[:, 0], s.requires_grad_()),
                 lambda: gated_scan_step(x[:, 0], x[:, 0], s.detach(), new_state=s.detach()[:, :5]),
                 lambda: gated_scan_step(x[:, 0], x[:, 0], torch.zeros(6, 2, device=cuda).t())):
        with pytest.raises(RuntimeError):
            call()
    y = x.clone().requires_grad_()
    out, _ = gated_scan(y, x)
    first, = torch.autograd.grad(out.square().sum(), y, create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative, and no silent zero
        first.sum().backward()


def test_module_runs_and_steps(cuda):
    from pulsartecture_b200 import GatedRecurrence

    torch.manual_seed(0)
    m = GatedRecurrence(48, 32).to(cuda)
    u = torch.randn(2, 20, 48, device=cuda)
    out, state = m(u, return_state=True)
    out.sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
    s = m.init_state(2)
    steps = torch.stack([m.step(u[:, t], s) for t in range(20)], 1)
    assert torch.allclose(steps, out, rtol=1e-5, atol=1e-5) and torch.allclose(s, state, rtol=1e-5, atol=1e-5)
