"""float64 restatement of the gated recurrence and its gradient, with the
magnitudes that bound what rounding can do to them.

    h_t = a_t h_{t-1} + b_t

Any order of evaluation multiplies a contribution b_s by a_{s+1} ... a_t, each
factor and each product off by a few units u = 2^-24, and adds them up. With
M_t = |a_t| M_{t-1} + |b_t|, an evaluation whose every factor is off by at most
k u is within E_t = |a_t| E_{t-1} + k u M_t of h_t.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24


def coefficients(gate: torch.Tensor, act: str):
    g = gate.double()
    if act == "sigmoid":
        return torch.sigmoid(g), torch.sigmoid(-g)
    return g, 1 - g


def _walk(a, b, first):
    h, steps = first, []
    for t in range(a.shape[1]):
        h = a[:, t] * h + b[:, t]
        steps.append(h)
    return torch.stack(steps, 1)


def scan(x, gate, state=None, act="sigmoid", mix=True, k=8.0, dout=None, dstate=None):
    """(values, bounds): dicts of out, state and, given dout, dx, dgate, dstate."""
    a, rest = coefficients(gate, act)
    x = x.double()
    B, T, D = x.shape
    zero = torch.zeros(B, D, dtype=torch.float64)
    h0 = zero if state is None else state.double()
    b = rest * x if mix else x
    h = _walk(a, b, h0)
    M = _walk(a.abs(), b.abs(), h0.abs())
    E = _walk(a.abs(), k * U * M, zero)
    val = {"out": h, "state": h[:, -1]}
    bound = {"out": E, "state": E[:, -1]}
    if dout is not None:
        d = dout.double().clone()
        if dstate is not None:
            d[:, -1] += dstate.double()
        # r_t = a_t G_t is carried to token t - 1: G_t = d_t + r_{t+1}
        shift = lambda v: torch.cat([v[:, 1:], torch.zeros_like(v[:, :1])], 1).flip(1)  # noqa: E731
        G = _walk(shift(a), d.flip(1), zero).flip(1)
        N = _walk(shift(a.abs()), d.abs().flip(1), zero).flip(1)
        F = _walk(shift(a.abs()), k * U * N.flip(1), zero).flip(1)
        before = torch.cat([h0[:, None], h[:, :-1]], 1)
        Eb = torch.cat([zero[:, None], E[:, :-1]], 1)
        inner = before - x if mix else before
        inner_err = Eb + U * (before.abs() + x.abs())
        c = rest.abs() if mix else torch.ones_like(a)
        val["dx"] = G * rest if mix else G
        bound["dx"] = c * (F + k * U * G.abs())
        da = G * inner
        s = a * rest if act == "sigmoid" else torch.ones_like(a)
        val["dgate"] = da * s
        bound["dgate"] = s.abs() * (F * inner.abs() + (G.abs() + F) * inner_err + 2 * k * U * da.abs())
        val["dstate"] = a[:, 0] * G[:, 0]
        bound["dstate"] = a[:, 0].abs() * (F[:, 0] + k * U * G[:, 0].abs())
    return val, bound
