"""The recurrence and vocabulary-row operators as cases to be timed and compared.

Three operators, each in its plain form (elementary torch operations, fp32)
and as the calls of this package:

  recur    h_t = a_t h_{t-1} + b_t per channel, a = sigmoid(gate) or gate,
           b = (1 - a) x or x: forward, backward, and one token
  logprob  the log probability of a given token in each row of logits, the
           row's entropy and its most probable tokens: forward, backward
  distill  the KL divergence from a teacher known by its largest logits to
           each row of logits: forward, backward

`own` picks the side; inputs come from the seed alone.
"""
import math

import torch

own = False

F32, BF16 = "float32", "bfloat16"


def listed():
    return [
        # one token for a full decode batch (32 heads of 128 channels)
        dict(name="recur step", op="recur", kind="step", batch=256, length=1, width=4096, dtype=BF16,
             gate_act="sigmoid", mix=True, state=True),
        # prompts of a batch (16 heads of 128 channels)
        dict(name="recur prefill", op="recur", kind="forward", batch=8, length=4096, width=2048, dtype=BF16,
             gate_act="sigmoid", mix=True, state=False),
        # one long document continued from a kept state
        dict(name="recur long", op="recur", kind="forward", batch=1, length=65536, width=4096, dtype=BF16,
             gate_act="sigmoid", mix=True, state=True),
        # a training step of the language model's recurrent layer
        dict(name="recur train", op="recur", kind="train", batch=16, length=2048, width=1024, dtype=BF16,
             gate_act="sigmoid", mix=True, state=False),
        # ragged sizes, decay factors given as they are, gradients into the initial state
        dict(name="recur odd", op="recur", kind="train", batch=3, length=1001, width=515, dtype=F32,
             gate_act="identity", mix=False, state=True),
        # sampled tokens of a decode batch with their alternatives, some tokens forbidden
        dict(name="logprob decode", op="logprob", kind="forward", batch=1, length=64, vocab=32000, dtype=BF16,
             top_k=20, temperature=1.0, shifted=False, masked=True),
        # scoring a batch of documents
        dict(name="logprob score", op="logprob", kind="forward", batch=4, length=2048, vocab=32000, dtype=BF16,
             top_k=5, temperature=1.0, shifted=False, masked=False),
        # next-token loss with an entropy term: the last position of a sequence has no target
        dict(name="logprob train", op="logprob", kind="train", batch=4, length=2048, vocab=32000, dtype=BF16,
             top_k=0, temperature=1.0, shifted=True, masked=False),
        # a vocabulary whose rows start off any 16-byte boundary, sharpened, many alternatives
        dict(name="logprob odd", op="logprob", kind="forward", batch=1, length=301, vocab=50257, dtype=F32,
             top_k=32, temperature=0.7, shifted=False, masked=False),
        # distillation with the rest of the vocabulary as one more class
        dict(name="distill train", op="distill", kind="train", rows=4096, vocab=32000, dtype=BF16, entries=64,
             temperature=1.0, tail=True, padded=False),
        # few teacher entries, some rows with fewer, softened, ragged vocabulary
        dict(name="distill odd", op="distill", kind="train", rows=257, vocab=50257, dtype=BF16, entries=17,
             temperature=2.0, tail=False, padded=True),
        # watching the divergence of a few positions
        dict(name="distill small", op="distill", kind="forward", rows=8, vocab=32000, dtype=F32, entries=8,
             temperature=1.0, tail=True, padded=False),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["recur", "logprob", "distill"])
    dtype = rng.choice([BF16, BF16, F32])
    if op == "recur":
        kind = rng.choice(["step", "forward", "train"])
        width = _spread(rng, 64, 4096)
        width = width if rng.random() < 0.4 else max(64, width // 64 * 64)
        if kind == "step":
            batch, length = _spread(rng, 1, 512), 1
        else:
            batch = _spread(rng, 1, 16)
            length = _spread(rng, 1, min(65536, max(2, (1 << 25) // (batch * width))))
        return dict(op=op, kind=kind, batch=batch, length=length, width=width, dtype=dtype,
                    gate_act=rng.choice(["sigmoid", "sigmoid", "identity"]), mix=rng.random() < 0.7,
                    state=kind == "step" or rng.random() < 0.5)
    vocab = _spread(rng, 1000, 131072)
    vocab = vocab if rng.random() < 0.4 else vocab // 8 * 8
    rows = _spread(rng, 1, max(2, min(8192, (1 << 27) // vocab)))
    kind = rng.choice(["forward", "train"])
    temperature = rng.choice([1.0, 1.0, 0.7, 2.0])
    if op == "logprob":
        batch = rng.choice([1, 1, 2, 3])
        return dict(op=op, kind=kind, batch=batch, length=max(2, rows // batch), vocab=vocab, dtype=dtype,
                    top_k=rng.choice([0, 1, 5, 20, 32]), temperature=temperature, shifted=rng.random() < 0.4,
                    masked=rng.random() < 0.3)
    return dict(op=op, kind=kind, rows=rows, vocab=vocab, dtype=dtype, entries=_spread(rng, 1, 128),
                temperature=temperature, tail=rng.random() < 0.5, padded=rng.random() < 0.4)


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = getattr(torch, case["dtype"])

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev) * scale

    if case["op"] == "recur":
        B, T, D = case["batch"], case["length"], case["width"]
        lead = (B, D) if case["kind"] == "step" else (B, T, D)
        s = dict(case=case, x=normal(*lead).to(dt), state=normal(B, D) if case["state"] else None)
        # gates that forget over tens to thousands of tokens
        gate = normal(*lead, scale=2.0) + 3.0
        s["gate"] = (gate if case["gate_act"] == "sigmoid" else torch.sigmoid(gate)).to(dt)
        if case["kind"] == "step":
            s["new_state"] = torch.empty_like(s["state"])
        if case["kind"] == "train":
            s["dout"], s["dstate"] = normal(*lead).to(dt), normal(B, D)
            for n in ("x", "gate") + (("state",) if case["state"] else ()):
                s[n].requires_grad_()
        return s
    V = case["vocab"]
    if case["op"] == "logprob":
        B, T = case["batch"], case["length"]
        logits = normal(B, T, V, scale=2.5)
        if case["masked"]:  # a padded end of the vocabulary, and tokens that a grammar forbids in half of the rows
            logits[..., V - V // 50:] = -math.inf
            forbidden = torch.rand(B, T, V, generator=g, device=dev) < 0.3
            forbidden[:, ::2] = False
            logits.masked_fill_(forbidden, -math.inf)
        logits = logits.to(dt)
        # tokens as they are sampled: likely ones more often
        targets = torch.argmax(logits[..., :V - V // 50].float() / 2.5 + 3.0 * torch.rand(B, T, 1, generator=g, device=dev)
                               * normal(B, T, V - V // 50), dim=-1)
        targets[torch.rand(B, T, generator=g, device=dev) < 0.05] = -100  # padding
        train = case["kind"] == "train"
        if case["shifted"]:  # row t of a sequence is given its token t + 1
            targets = torch.cat([targets[:, 1:], torch.full_like(targets[:, :1], -100)], 1) if train else targets[:, 1:].contiguous()
        s = dict(case=case, logits=logits, targets=targets)
        if train:
            logits.requires_grad_()
            s["dlogprobs"], s["dentropy"] = normal(B, T), normal(B, T, scale=0.01)
            if case["shifted"]:
                s["dentropy"][:, -1] = 0
            if case["top_k"]:
                s["dtop"] = normal(B, T, case["top_k"], scale=0.1)
        return s
    rows, K = case["rows"], case["entries"]
    teacher = normal(rows, V, scale=3.0)
    logits = (0.8 * teacher + normal(rows, V)).to(dt)  # a student on its way to the teacher
    top, ids = torch.topk(teacher, K, dim=-1)
    s = dict(case=case, logits=logits, teacher_ids=ids, teacher_logits=top, teacher_lse=None)
    if case["tail"]:
        s["teacher_lse"] = torch.logsumexp(teacher / case["temperature"], dim=-1)
    if case["padded"]:  # rows for which fewer entries were kept, a few with none
        kept = torch.randint(0, K + 1, (rows, 1), generator=g, device=dev)
        s["teacher_ids"] = torch.where(torch.arange(K, device=dev) < kept, ids, -1)
    if case["kind"] == "train":
        logits.requires_grad_()
        s["dloss"] = normal(rows)
    return s


# ----------------------------------------------------------------------------- recur, plain
def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t from h = 0 along dim 1, by doubling."""
    d = 1
    while d < a.shape[1]:
        b = torch.cat([b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return b


def _coefficients(case, gate):
    """(a, 1 - a) in 32 bits."""
    gate = gate.detach().float()
    if case["gate_act"] == "sigmoid":
        return torch.sigmoid(gate), torch.sigmoid(-gate)
    return gate, 1.0 - gate


def _recur_plain(s):
    case, x, dt = s["case"], s["x"].detach().float(), s["x"].dtype
    a, rest = _coefficients(case, s["gate"])
    state = None if s["state"] is None else s["state"].detach()
    b = rest * x if case["mix"] else x
    if case["kind"] == "step":
        h = a * state + b
        return {"out": h.to(dt), "state": h}
    first = b[:, :1] if state is None else b[:, :1] + a[:, :1] * state[:, None]
    h = _scan(a, torch.cat([first, b[:, 1:]], 1))
    got = {"out": h.to(dt), "state": h[:, -1].clone()}
    if case["kind"] == "train":
        dout = s["dout"].float()
        dout = torch.cat([dout[:, :-1], dout[:, -1:] + s["dstate"][:, None]], 1)
        after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
        G = _scan(after.flip(1), dout.flip(1)).flip(1)
        before = torch.cat([torch.zeros_like(h[:, :1]) if state is None else state[:, None], h[:, :-1]], 1)
        da = G * (before - x) if case["mix"] else G * before
        got["dx"] = (G * rest if case["mix"] else G).to(dt)
        got["dgate"] = (da * a * rest if case["gate_act"] == "sigmoid" else da).to(dt)
        if state is not None:
            got["dstate"] = a[:, 0] * G[:, 0]
    return got


# ----------------------------------------------------------------------------- logprob, plain
def _log_softmax(z, temperature):
    """Over the last dimension, in z's type; a row with nothing but -inf gives -inf."""
    m = z.amax(-1, keepdim=True)
    z = (z - torch.where(m == -math.inf, 0.0, m)) * (1.0 / temperature)
    total = torch.exp(z).sum(-1, keepdim=True)
    return z - torch.where(total == 0, 0.0, torch.log(total))


def _order(x):
    """Whole numbers in the order of the 32-bit values of x, then of the lower index first."""
    bits = x.view(torch.int32).to(torch.int64)
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    return bits * (1 << 31) + (x.shape[-1] - 1 - torch.arange(x.shape[-1], device=x.device))


def _rows(s):
    """The logits that have a target: scored sequences leave out their last row, trained ones mark it in the targets."""
    cut = s["case"]["shifted"] and s["case"]["kind"] == "forward"
    return s["logits"][:, :-1] if cut else s["logits"]


def _logprob_plain(s):
    case = s["case"]
    logits = _rows(s).detach()
    z, targets, k = logits.float(), s["targets"], case["top_k"]
    lp = _log_softmax(z, case["temperature"])
    p = torch.exp(lp)
    counted = targets != -100
    at = torch.where(counted, targets, 0)[..., None]
    got = {"logprobs": torch.where(counted, lp.gather(-1, at)[..., 0], 0.0)}
    plogp = torch.where(p > 0, p * lp, 0.0)
    got["entropy"] = -plogp.sum(-1)
    if k:
        got["top_ids"] = torch.topk(_order(z), k, dim=-1).indices
        got["top_logprobs"] = lp.gather(-1, got["top_ids"])
    if case["kind"] == "train":
        w = torch.where(counted, s["dlogprobs"], 0.0)[..., None]
        total = w
        dz = torch.zeros_like(z).scatter_add_(-1, at, w)
        if k:
            dz.scatter_add_(-1, got["top_ids"], s["dtop"])
            total = total + s["dtop"].sum(-1, keepdim=True)
        dz = dz - total * p - s["dentropy"][..., None] * (plogp + p * got["entropy"][..., None])
        got["dlogits"] = (dz / case["temperature"]).to(logits.dtype)
    return got


# ----------------------------------------------------------------------------- distill, plain
def _distill_plain(s):
    case, T = s["case"], s["case"]["temperature"]
    logits = s["logits"].detach()
    lp = _log_softmax(logits.float(), T)
    p = torch.exp(lp)
    valid = s["teacher_ids"] >= 0
    at = torch.where(valid, s["teacher_ids"], 0)
    t = torch.where(valid, s["teacher_logits"], -math.inf)
    some = valid.any(-1)
    if case["tail"]:
        lq = t * (1.0 / T) - s["teacher_lse"][:, None]
    else:
        lq = _log_softmax(t, T)
    q = torch.exp(lq)
    loss = torch.where(q > 0, q * (lq - lp.gather(-1, at)), 0.0).sum(-1)
    mass = q.sum(-1)
    if case["tail"]:
        member = torch.zeros_like(lp).scatter_reduce_(-1, at, valid.float(), "amax") > 0
        p_rest = torch.where(member, 0.0, p).sum(-1)
        q_rest = torch.where(some, (1.0 - mass).clamp_min(0.0), 0.0)
        rest = torch.where(q_rest > 0, q_rest / p_rest, 0.0)
        loss = loss + torch.where(q_rest > 0, q_rest * torch.log(rest), 0.0)
        mass = mass + q_rest
    got = {"loss": loss}
    if case["kind"] == "train":
        dz = p * mass[:, None]
        if case["tail"]:
            dz = dz - torch.where(member, 0.0, p * rest[:, None])
        dz.scatter_add_(-1, at, -q)
        got["dlogits"] = (dz * (s["dloss"] / T)[:, None]).to(logits.dtype)
    return got


# ----------------------------------------------------------------------------- this package's calls
def _recur_own(s):
    from pulsartecture_b200 import gated_scan, gated_scan_step

    case = s["case"]
    how = dict(gate_act=case["gate_act"], mix=case["mix"])
    if case["kind"] == "step":
        out, state = gated_scan_step(s["x"], s["gate"], s["state"], new_state=s["new_state"], **how)
        return {"out": out, "state": state}
    out, state = gated_scan(s["x"], s["gate"], s["state"], return_state=True, **how)
    got = {"out": out.detach(), "state": state.detach()}
    if case["kind"] == "train":
        names = ["x", "gate"] + (["state"] if case["state"] else [])
        grads = torch.autograd.grad([out, state], [s[n] for n in names], [s["dout"], s["dstate"]])
        got.update({"d" + n: v for n, v in zip(names, grads)})
    return got


def _logprob_own(s):
    from pulsartecture_b200 import token_logprobs

    case = s["case"]
    r = token_logprobs(_rows(s), s["targets"], top_k=case["top_k"], temperature=case["temperature"])
    got = {"logprobs": r.logprobs.detach(), "entropy": r.entropy.detach()}
    if case["top_k"]:
        got.update(top_ids=r.top_ids, top_logprobs=r.top_logprobs.detach())
    if case["kind"] == "train":
        outs, given = [r.logprobs, r.entropy], [s["dlogprobs"], s["dentropy"]]
        if case["top_k"]:
            outs, given = outs + [r.top_logprobs], given + [s["dtop"]]
        got["dlogits"], = torch.autograd.grad(outs, [s["logits"]], given)
    return got


def _distill_own(s):
    from pulsartecture_b200 import distill_topk

    case = s["case"]
    loss = distill_topk(s["logits"], s["teacher_ids"], s["teacher_logits"], s["teacher_lse"],
                        temperature=case["temperature"])
    got = {"loss": loss.detach()}
    if case["kind"] == "train":
        got["dlogits"], = torch.autograd.grad([loss], [s["logits"]], [s["dloss"]])
    return got


def run(state):
    op = state["case"]["op"]
    if own:
        return {"recur": _recur_own, "logprob": _logprob_own, "distill": _distill_own}[op](state)
    return {"recur": _recur_plain, "logprob": _logprob_plain, "distill": _distill_plain}[op](state)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = 4 if case["dtype"] == F32 else 2
    train = case["kind"] == "train"
    if case["op"] == "recur":
        n, c = case["batch"] * case["length"] * case["width"], case["batch"] * case["width"]
        moved = 3 * n * e + 4 * c * (2 if case["state"] else 1)
        if train:  # dout in, dx and dgate out; the state's gradients
            moved += 3 * n * e + 4 * c * (2 if case["state"] else 1)
        return {"bytes": moved, "flops": n * (22 if train else 8)}
    if case["op"] == "logprob":
        rows = case["batch"] * (case["length"] - (1 if case["shifted"] and not train else 0))
        n, extra = rows * case["vocab"], rows * (16 + 12 * case["top_k"])
        if train:
            return {"bytes": 2 * n * e + 2 * extra, "flops": 14 * n}
        return {"bytes": n * e + extra, "flops": 7 * n}
    n, extra = case["rows"] * case["vocab"], case["rows"] * (8 + 12 * case["entries"])
    return {"bytes": n * e * (2 if train else 1) + extra, "flops": n * (10 if train else 6)}


# ----------------------------------------------------------------------------- from the definitions, in 64 bits
def _recur_exact(s):
    case = s["case"]
    x, gate = s["x"].detach().double(), s["gate"].detach().double()
    if case["kind"] == "step":
        x, gate = x[:, None], gate[:, None]
    a = 1 / (1 + torch.exp(-gate)) if case["gate_act"] == "sigmoid" else gate
    b = (1 - a) * x if case["mix"] else x
    B, T, D = x.shape
    h0 = torch.zeros_like(x[:, 0]) if s["state"] is None else s["state"].detach().double()
    past = torch.empty(T + 1, B, D, dtype=torch.float64, device=x.device)
    past[0] = h0
    for t in range(T):
        torch.addcmul(b[:, t], a[:, t], past[t], out=past[t + 1])
    if case["kind"] == "step":
        return {"out": past[1], "state": past[1]}
    got = {"out": past[1:].transpose(0, 1), "state": past[T]}
    if case["kind"] == "train":
        dout = s["dout"].double()
        G = torch.empty_like(past[1:])
        carry = s["dstate"].double()
        for t in reversed(range(T)):
            torch.add(dout[:, t], carry, out=G[t])
            carry = G[t] * a[:, t]
        G = G.transpose(0, 1)
        da = G * past[:-1].transpose(0, 1)
        if case["mix"]:
            da = da - G * x
        got["dx"] = G * (1 - a) if case["mix"] else G
        got["dgate"] = da * a * (1 - a) if case["gate_act"] == "sigmoid" else da
        if s["state"] is not None:
            got["dstate"] = carry
    return got


def _logprob_exact(s):
    case = s["case"]
    every = _rows(s).detach()
    found = {}
    for i in range(every.shape[0]):
        z = every[i].double() / case["temperature"]
        lse = torch.logsumexp(z, -1, keepdim=True)
        p = torch.exp(z - lse)
        lp = z - lse
        target = s["targets"][i]
        on = (target != -100).double()
        at = target.clamp_min(0)[:, None]
        part = {"logprobs": torch.where(on > 0, lp.gather(-1, at)[:, 0], 0.0)}
        part["entropy"] = torch.special.entr(p).sum(-1)
        if case["top_k"]:
            part["top_logprobs"] = torch.topk(lp, case["top_k"], dim=-1).values
        if case["kind"] == "train":
            w = s["dlogprobs"][i].double() * on
            H = part["entropy"][:, None]
            dz = -p * w[:, None] - s["dentropy"][i].double()[:, None] * (p * H - torch.special.entr(p))
            dz.scatter_add_(-1, at, w[:, None])
            if case["top_k"]:
                # the k largest, the lower index first among equals, as in a stable sort
                ids = torch.sort(every[i].float(), dim=-1, descending=True, stable=True).indices[:, :case["top_k"]]
                d = s["dtop"][i].double()
                dz.scatter_add_(-1, ids, d)
                dz -= p * d.sum(-1, keepdim=True)
            part["dlogits"] = dz / case["temperature"]
        for n, v in part.items():
            found.setdefault(n, []).append(v)
    got = {n: torch.stack(v) for n, v in found.items()}
    if case["top_k"]:
        got["top_ids"] = None
    return got


def _distill_exact(s):
    case, T = s["case"], s["case"]["temperature"]
    z = s["logits"].detach().double() / T
    valid = s["teacher_ids"] >= 0
    at = s["teacher_ids"].clamp_min(0)
    t = s["teacher_logits"].double() / T
    t[~valid] = -math.inf
    if case["tail"]:
        q = torch.exp(t - s["teacher_lse"].double()[:, None])
    else:
        top = torch.where(valid.any(-1), t.amax(-1), 0.0)[:, None]
        q = torch.exp(t - top)
        q = q / q.sum(-1, keepdim=True).clamp_min(1e-300)
    lse = torch.logsumexp(z, -1)
    loss = (torch.xlogy(q, q) - torch.where(valid, q * (z.gather(-1, at) - lse[:, None]), 0.0)).sum(-1)
    mass = q.sum(-1)
    p = torch.exp(z - lse[:, None])
    dz = None
    if case["tail"]:
        rest = z.clone()
        row = torch.arange(z.shape[0], device=z.device)[:, None].expand_as(at)
        rest[row[valid], at[valid]] = -math.inf
        lrest = torch.logsumexp(rest, -1)
        q_rest = (1 - mass).clamp_min(0) * valid.any(-1)
        loss = loss + torch.xlogy(q_rest, q_rest) - q_rest * (lrest - lse)
        mass = mass + q_rest
        if case["kind"] == "train":
            dz = p * mass[:, None] - torch.exp(rest - lrest[:, None]) * q_rest[:, None]
    got = {"loss": loss}
    if case["kind"] == "train":
        dz = p * mass[:, None] if dz is None else dz
        dz.scatter_add_(-1, at, -q)
        got["dlogits"] = dz * s["dloss"].double()[:, None] / T
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"recur": _recur_exact, "logprob": _logprob_exact, "distill": _distill_exact}[case["op"]](s)
