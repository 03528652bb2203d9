"""The two halves of a residual layer that is trained, as a user's program calls
them: the gated linear recurrence over time (forward, with its gradient, and one
token at a time) and the gated feed-forward product over the channels (forward, with
its gradient, and for the few tokens of a decode step).

listed() names the cases, draw() gives more of the same ranges, prepare() makes
what the program holds before the call, run() is one pass (the plain form, or
with ``own`` the framework's operators), work() the bytes and operations a pass
cannot do without, exact() the results in 64 bits.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
SIZE = {"bf16": 2, "f32": 4}
GELU = math.sqrt(2.0 / math.pi), 0.044715


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _ops():
    """The framework's entry points (only where own is true)."""
    pkg = os.path.join(_ROOT, "mamba2-jax-pallas_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from mamba2_jax import ops
    return ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _glu(kind, tokens, dim, hidden, dtype, activation):
    return dict(kind=kind, tokens=tokens, dim=dim, hidden=hidden, dtype=dtype, activation=activation)


def _rec(kind, batch, seqlen, dim, dtype, fused, packed, carried):
    """fused: x and the two gates are slices of one projection's output.  packed: the mean
    length of the sequences that share a row, the last of them followed by padding (0: one
    sequence a row).  carried: the rows go on from states, and theirs are returned."""
    return dict(kind=kind, batch=batch, seqlen=seqlen, dim=dim, dtype=dtype, fused=fused, packed=packed,
                carried=carried)


def listed():
    named = [
        # the feed-forward product of one token of one request: the weights' bytes, launch latency
        ("glu_step", _glu("glu", 1, 2560, 6912, "bf16", "silu")),
        # of a decode step of sixteen requests
        ("glu_step_16", _glu("glu", 16, 2560, 6912, "bf16", "silu")),
        # of a 4096-token prompt
        ("glu_prompt", _glu("glu", 4096, 2560, 6912, "bf16", "silu")),
        # a training step's, a packed batch
        ("glu_train", _glu("glu_train", 8192, 2560, 6912, "bf16", "silu")),
        # a ragged batch, a width and a hidden size that no tile divides
        ("glu_train_odd", _glu("glu_train", 333, 1001, 1365, "bf16", "gelu")),
        # a small model in float32
        ("glu_train_f32", _glu("glu_train", 1024, 768, 2048, "f32", "gelu")),
        # one token of sixteen requests: launch latency
        ("rec_step", _rec("rec_step", 16, 1, 2560, "bf16", True, 0, True)),
        # a long prompt: few channels, many steps
        ("rec_prompt", _rec("rec", 1, 16384, 2560, "bf16", True, 0, True)),
        # a training batch, many channels
        ("rec_train", _rec("rec_train", 8, 2048, 5120, "bf16", False, 0, False)),
        # documents packed into one long row, with padding behind the last
        ("rec_train_packed", _rec("rec_train", 1, 8191, 2560, "bf16", True, 700, False)),
        # a ragged batch of a width that no vector divides, going on from states
        ("rec_train_odd", _rec("rec_train", 3, 777, 1001, "bf16", False, 0, True)),
        # a small model in float32
        ("rec_train_f32", _rec("rec_train", 4, 1024, 768, "f32", False, 300, True)),
    ]
    return [dict(c, name=n) for n, c in named]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    d = _log_int(rng, lo, hi)
    if rng.random() < 0.6:                      # widths of models are mostly round, not always
        d = max(lo, d // 64 * 64)
    return d


def draw(rng):
    kind = rng.choice(["glu", "glu_train", "glu_train", "rec_step", "rec", "rec_train", "rec_train"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind in ("glu", "glu_train"):
        tokens, dim, hidden = _log_int(rng, 1, 8192), _width(rng, 64, 4096), _width(rng, 64, 8192)
        cap = 8192 * 2560 * 6912 // (8 if dtype == "f32" else 1)
        while tokens * dim * hidden > cap:
            tokens //= 2
        return _glu(kind, tokens, dim, hidden, dtype, rng.choice(["silu", "gelu"]))
    batch, dim = _log_int(rng, 1, 64 if kind == "rec_step" else 16), _width(rng, 16, 5120)
    fused = rng.random() < 0.5
    if kind == "rec_step":
        return _rec(kind, batch, 1, dim, dtype, fused, 0, True)
    seqlen = _log_int(rng, 1, 16384)
    while batch * seqlen * dim > 8 * 2048 * 5120:
        batch, seqlen = max(1, batch // 2), seqlen if batch > 1 else seqlen // 2
    packed = _log_int(rng, 2, 2000) if rng.random() < 0.4 else 0
    return _rec(kind, batch, seqlen, dim, dtype, fused, packed, rng.random() < 0.5)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + 29)


def _randn(shape, g, dt, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dt)


def _seq_idx(case, g):
    """Sequences of random lengths behind each other in every row, about a twentieth of
    the row padding (-1) at its end."""
    b, n = case["batch"], case["seqlen"]
    starts = torch.rand((b, n), generator=g, device=DEV) < 1.0 / case["packed"]
    idx = starts.cumsum(1).int()
    kept = torch.randint(n - n // 10, n + 1, (b, 1), generator=g, device=DEV)
    return torch.where(torch.arange(n, device=DEV)[None] < kept, idx, torch.full_like(idx, -1))


def prepare(case, seed):
    g = _gen(seed)
    dt = _dtype(case)
    kind, d = case["kind"], case["dim"]
    if kind in ("glu", "glu_train"):
        n, f = case["tokens"], case["hidden"]
        # what a norm leaves, and weights that keep the products at the order of one
        x = _randn((n, d), g, dt)
        w = _randn((2 * f, d), g, dt, 1.0 / math.sqrt(d))
        state = dict(case=case, x=x, w=w)
        if kind == "glu_train":
            state["dh"] = _randn((n, f), g, dt, 0.01)
            x.requires_grad_()
            w.requires_grad_()
        return state
    b, n = case["batch"], case["seqlen"]
    shape = (b, d) if kind == "rec_step" else (b, n, d)
    if case["fused"]:
        parts = _randn((*shape[:-1], 3 * d), g, dt).split(d, dim=-1)
        x, r, i = (p.detach() for p in parts)
    else:
        x, r, i = (_randn(shape, g, dt) for _ in range(3))
    # a state's memory at an open gate: from 2 to 1000 steps
    A = -torch.exp(torch.empty(d, device=DEV).uniform_(math.log(1e-3), math.log(0.5), generator=g))
    state = dict(case=case, x=x, r=r, i=i, A=A, h0=None, seq=None)
    if case["carried"]:
        state["h0"] = torch.randn((b, d), generator=g, device=DEV)
    if case["packed"]:
        state["seq"] = _seq_idx(case, g)
    if kind == "rec_train":
        state["dh"] = _randn(shape, g, dt, 0.01)
        leaves = [x, r, i, A]
        if case["carried"]:
            state["dlast"] = torch.randn((b, d), generator=g, device=DEV) * 0.01
            leaves.append(state["h0"])
        for t in leaves:
            t.requires_grad_()
        state["leaves"] = leaves
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _run_own(state):
    ops = _ops()
    case = state["case"]
    kind = case["kind"]
    if kind == "glu":
        return ops.gated_linear(state["x"], state["w"], activation=case["activation"])
    if kind == "glu_train":
        h = ops.gated_linear(state["x"], state["w"], activation=case["activation"])
        dx, dw = torch.autograd.grad(h, (state["x"], state["w"]), state["dh"])
        return dict(h=h.detach(), dx=dx, dw=dw)
    if kind == "rec_step":
        last, y = ops.gated_linear_recurrence_update(state["h0"], state["x"], state["r"], state["i"], state["A"])
        return dict(y=y, last=last)
    out = ops.gated_linear_recurrence(state["x"], state["r"], state["i"], state["A"], initial_states=state["h0"],
                                      seq_idx=state["seq"], return_final_states=case["carried"])
    h, last = out if case["carried"] else (out, None)
    if kind == "rec":
        return dict(h=h, last=last) if case["carried"] else dict(h=h)
    ups = ((h, last), (state["dh"], state["dlast"])) if case["carried"] else ((h,), (state["dh"],))
    grads = torch.autograd.grad(ups[0], state["leaves"], ups[1])
    got = dict(h=h.detach(), **dict(zip(("dx", "dr", "di", "dA", "dh0"), grads)))
    if case["carried"]:
        got["last"] = last.detach()
    return got


def _act(z, activation):
    """(act(z), act'(z))"""
    if activation == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    c, k = GELU
    t = torch.tanh(c * (z + k * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * k * z * z)


def _gates(state):
    """(q, s, log a, sqrt(1 - a^2), what is added to the state, positions that clear it and
    positions that are padding: both (batch, seqlen, 1), or None)"""
    q, s = torch.sigmoid(state["r"].float()), torch.sigmoid(state["i"].float())
    la = state["A"] * q
    beta = torch.sqrt(-torch.expm1(2 * la))
    seq, clear, pad = state["seq"], None, None
    if seq is not None:
        pad = (seq < 0)[..., None]
        clear = torch.zeros_like(pad)
        clear[:, 1:, 0] = (seq[:, 1:] != seq[:, :-1]) & (seq[:, 1:] >= 0)
    return q, s, la, beta, beta * s * state["x"].float(), clear, pad


def _decays(la, add, clear, pad):
    a = torch.exp(la)
    if clear is not None:
        zero = torch.zeros_like(a)
        a = torch.where(pad, torch.ones_like(a), torch.where(clear, zero, a))
        add = torch.where(pad, zero, add)
    return a, add


def _plain_rec(state):
    """-> (h as it is carried, the final state, the gates, the decays)"""
    gates = _gates(state)
    a, add = _decays(gates[2], gates[4], gates[5], gates[6])
    b, n, d = add.shape
    h = torch.empty_like(add)
    at = state["h0"].float() if state["h0"] is not None else torch.zeros((b, d), device=DEV)
    for av, bv, hv in zip(a.unbind(1), add.unbind(1), h.unbind(1)):
        at = torch.addcmul(bv, av, at, out=hv)
    return h, at, gates, a


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    kind = case["kind"]
    dt = _dtype(case)
    with torch.no_grad():
        if kind in ("glu", "glu_train"):
            x, w = state["x"].float(), state["w"].float()
            g, v = (x @ w.t()).chunk(2, dim=1)
            act, slope = _act(g, case["activation"])
            h = (act * v).to(dt)
            if kind == "glu":
                return h
            dh = state["dh"].float()
            dz = torch.cat([dh * v * slope, dh * act], dim=1)
            return dict(h=h, dx=(dz @ w).to(dt), dw=(dz.t() @ x).to(dt))
        if kind == "rec_step":
            _, _, la, _, add, _, _ = _gates(state)
            last = torch.exp(la) * state["h0"] + add
            return dict(y=last.to(dt), last=last)
        h, last, (q, s, la, beta, add, clear, pad), a = _plain_rec(state)
        hidden = h if pad is None else torch.where(pad, torch.zeros_like(h), h)
        got = dict(h=hidden.to(dt))
        if case["carried"]:
            got["last"] = last.clone()
        if kind == "rec":
            return got
        up = state["dh"].float()
        if pad is not None:
            up = torch.where(pad, torch.zeros_like(up), up)
        lam = torch.empty_like(up)
        at = state["dlast"] if case["carried"] else torch.zeros_like(last)
        for av, uv, lv in zip(reversed(a.unbind(1)), reversed(up.unbind(1)), reversed(lam.unbind(1))):
            torch.add(uv, at, out=lv)
            at = av * lv
        x = state["x"].float()
        before = torch.empty_like(h)
        before[:, 1:] = h[:, :-1]
        before[:, 0] = state["h0"] if state["h0"] is not None else 0.0
        if clear is not None:
            before = torch.where(clear, torch.zeros_like(before), before)
            lam = torch.where(pad, torch.zeros_like(lam), lam)
        ea = torch.exp(la)
        rise = torch.where(beta > 0, ea * ea / beta, torch.zeros_like(beta))
        dla = lam * (ea * before - rise * s * x)
        got.update(dx=(lam * beta * s).to(dt), di=(lam * beta * x * s * (1 - s)).to(dt),
                   dr=(dla * la * (1 - q)).to(dt), dA=(dla * q).sum((0, 1), dtype=torch.float64).float())
        if case["carried"]:
            got["dh0"] = at
        return got


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    es, d = SIZE[case["dtype"]], case["dim"]
    kind = case["kind"]
    if kind in ("glu", "glu_train"):
        n, f = case["tokens"], case["hidden"]
        forward = es * (n * d + 2 * f * d + n * f)
        if kind == "glu":
            return {"bytes": forward, "flops": 4 * n * f * d}
        # and the upstream gradient, dx and dw
        return {"bytes": forward + es * (n * f + n * d + 2 * f * d), "flops": 12 * n * f * d}
    rows = case["batch"] * case["seqlen"]
    other = 4 * d + (8 * case["batch"] * d if case["carried"] else 0) + (4 * rows if case["packed"] else 0)
    if kind != "rec_train":
        return {"bytes": 4 * rows * d * es + other, "flops": 20 * rows * d}
    # and the upstream gradients, those of x, the gates, A and the initial states
    other += 4 * d + (8 * case["batch"] * d if case["carried"] else 0)
    return {"bytes": 8 * rows * d * es + other, "flops": 60 * rows * d}


# ---------------------------------------------------------------------------
# the results in 64 bits
# ---------------------------------------------------------------------------
def _scan(a, b, dim):
    """y[t] = a[t] y[t - 1] + b[t] along dim, y[-1] = 0, by doubling spans (in place)."""
    n = a.shape[dim]
    span = 1
    while span < n:
        late, early = (lambda t: t.narrow(dim, span, n - span)), (lambda t: t.narrow(dim, 0, n - span))
        moved = late(a) * early(b)
        late(b).add_(moved)
        moved = late(a) * early(a)
        late(a).copy_(moved)
        span *= 2
    return b


def _exact_rec(state, case):
    train = case["kind"] == "rec_train"
    one = case["kind"] == "rec_step"
    x, r, i = (state[k].detach().double() for k in ("x", "r", "i"))
    if one:
        x, r, i = x[:, None], r[:, None], i[:, None]
    A = state["A"].detach().double()
    b, n, d = x.shape
    q, s = 1 / (1 + torch.exp(-r)), 1 / (1 + torch.exp(-i))
    la = A * q
    beta2 = -torch.expm1(2 * la)
    add = beta2.sqrt() * s * x
    a = torch.exp(la)
    live = torch.ones((b, n, 1), device=DEV, dtype=torch.float64)
    goes_on = live.clone()
    if state["seq"] is not None:
        seq = state["seq"].long()
        live = (seq >= 0).double()[..., None]
        goes_on[:, 1:] = ((seq[:, 1:] == seq[:, :-1]) | (seq[:, 1:] < 0)).double()[..., None]
        a = live * goes_on * a + (1 - live)
        add = add * live
    if state["h0"] is not None:
        h0 = state["h0"].detach().double()
        add = add.clone()
        add[:, 0] += a[:, 0] * h0
    h = _scan(a.clone(), add, 1)
    last = h[:, -1]
    if one:
        return dict(y=last, last=last)
    got = dict(h=h * live)
    if case["carried"]:
        got["last"] = last
    if not train:
        return got
    # the same recurrence from the end: each l[t] = up[t] + a[t + 1] l[t + 1]
    up = state["dh"].double() * live
    if case["carried"]:
        up[:, -1] += state["dlast"].double()
    later = torch.zeros_like(a)
    later[:, :-1] = a[:, 1:]
    lam = _scan(later.flip(1), up.flip(1), 1).flip(1)
    del later, up
    first = a[:, 0] * lam[:, 0]
    before = torch.zeros_like(h)
    before[:, 1:] = h[:, :-1]
    if case["carried"]:
        before[:, 0] = h0
    lam = lam * live
    got["dx"] = lam * beta2.sqrt() * s
    got["di"] = got["dx"] * x * (1 - s)
    ea2 = 1 - beta2
    dla = lam * (ea2.sqrt() * before * goes_on - (ea2 / beta2.sqrt()) * s * x)
    got["dr"] = dla * la * (1 - q)
    got["dA"] = (dla * q).sum((0, 1))
    if case["carried"]:
        got["dh0"] = first
    return got


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] not in ("glu", "glu_train"):
            return _exact_rec(state, case)
        n, d, f = case["tokens"], case["dim"], case["hidden"]
        w = state["w"].detach().double()
        train = case["kind"] == "glu_train"
        h = torch.empty((n, f), device=DEV, dtype=torch.float64)
        dx = torch.empty((n, d), device=DEV, dtype=torch.float64)
        dw = torch.zeros((2 * f, d), device=DEV, dtype=torch.float64)
        for part in torch.arange(n, device=DEV).split(1024):
            x = state["x"].detach()[part].double()
            g, v = x @ w[:f].t(), x @ w[f:].t()
            if case["activation"] == "silu":
                share = 1 / (1 + torch.exp(-g))
                slope = share + g * share * (1 - share)
            else:
                u = 2 * GELU[0] * (g + GELU[1] * g ** 3)
                share = 1 / (1 + torch.exp(-u))         # (1 + tanh(u / 2)) / 2
                slope = share + g * share * (1 - share) * 2 * GELU[0] * (1 + 3 * GELU[1] * g * g)
            h[part] = g * share * v
            if train:
                dh = state["dh"][part].double()
                dg, dv = dh * v * slope, dh * g * share
                dx[part] = dg @ w[:f] + dv @ w[f:]
                dw[:f] += dg.t().contiguous() @ x
                dw[f:] += dv.t().contiguous() @ x
        return dict(h=h, dx=dx, dw=dw) if train else h
