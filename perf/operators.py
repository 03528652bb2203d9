"""The operators on the vocabulary's side of training and scoring a language
model, as a user's program calls them: the loss of a linear head over the
vocabulary (with and without its gradient), the embedding lookup and its
gradient, and the clipping of a model's gradients by their global norm.

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
IGNORE = -100
CLIP_EPS = 1e-6
SIZE = {"bf16": 2, "f32": 4}


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
def _embed(tokens, vocab, dim, dtype, scaled):
    return dict(kind="embed", tokens=tokens, vocab=vocab, dim=dim, dtype=dtype, scaled=scaled)


def _embed_grad(tokens, vocab, dim, dtype, scaled, padding):
    return dict(kind="embed_grad", tokens=tokens, vocab=vocab, dim=dim, dtype=dtype, scaled=scaled,
                padding=padding)


def _loss(kind, tokens, vocab, dim, dtype, masked):
    """masked: the share of tokens (prompts, padding) that the loss leaves out."""
    return dict(kind=kind, tokens=tokens, vocab=vocab, dim=dim, dtype=dtype, masked=masked)


def _clip(layers, dim, vocab, dtype, max_norm):
    return dict(kind="clip", layers=layers, dim=dim, vocab=vocab, dtype=dtype, max_norm=max_norm)


def listed():
    named = [
        # the lookup of one decode step of sixteen requests (2.7b): launch latency
        ("embed_step", _embed(16, 50288, 2560, "bf16", False)),
        # the lookup of a packed training batch, with the sqrt(dim) scale some models apply
        ("embed_batch", _embed(16384, 50288, 2560, "bf16", True)),
        # its gradient, float32 parameters of the 130m model, unpadded vocabulary, a padding id
        ("embed_grad_130m", _embed_grad(2047, 50277, 768, "f32", False, True)),
        # its gradient for a packed batch of the 2.7b model
        ("embed_grad_batch", _embed_grad(16384, 50288, 2560, "bf16", True, False)),
        # scoring one candidate token after each of sixteen prompts: the head's weights read once
        ("score_step", _loss("score", 16, 50288, 2560, "bf16", 0.0)),
        # scoring a packed 4096-token prompt (perplexity)
        ("score_prompt", _loss("score", 4096, 50288, 2560, "bf16", 0.0)),
        # an instruction-tuning step of the 130m model: prompts left out of the loss
        ("train_130m", _loss("train", 2048, 50288, 768, "bf16", 0.4)),
        # the same in float32
        ("train_130m_f32", _loss("train", 1024, 50288, 768, "f32", 0.25)),
        # a ragged batch, vocabulary and width that no tile divides
        ("train_odd", _loss("train", 333, 32003, 1001, "bf16", 0.1)),
        # a packed pretraining batch of the 2.7b model
        ("train_large", _loss("train", 8192, 50288, 2560, "bf16", 0.0)),
        # float32 gradients of the 130m model, far above the bound
        ("clip_130m", _clip(24, 768, 50288, "f32", 1.0)),
        # bf16 gradients of the 1.3b model (float32 where the parameters are), below the bound
        ("clip_1b", _clip(48, 2048, 50288, "bf16", 1e5)),
    ]
    return [dict(c, name=n) for n, c in named]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["embed", "embed_grad", "embed_grad", "score", "train", "train", "clip"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "clip":
        layers, dim = rng.randint(1, 48), _log_int(rng, 64, 2048)
        vocab = _log_int(rng, 1000, 50288)
        return _clip(layers, dim, vocab, dtype, math.exp(rng.uniform(math.log(0.1), math.log(1e5))))
    vocab = _log_int(rng, 1000, 65536)
    dim = _log_int(rng, 64, 4096)
    if rng.random() < 0.6:                      # widths of models are mostly round, not always
        dim = max(64, dim // 64 * 64)
    if kind == "embed":
        tokens = _log_int(rng, 1, 16384)
        while tokens * dim > 16384 * 2560:
            tokens //= 2
        return _embed(tokens, vocab, dim, dtype, rng.random() < 0.5)
    if kind == "embed_grad":
        tokens = _log_int(rng, 1, 16384)
        while tokens * dim > 16384 * 2560:
            tokens //= 2
        while vocab * dim > 50288 * 2560:
            vocab //= 2
        return _embed_grad(tokens, vocab, dim, dtype, rng.random() < 0.5, rng.random() < 0.3)
    tokens = _log_int(rng, 1, 8192)
    cap = 8192 * 50288 * 2560 // (8 if dtype == "f32" else 1)
    while tokens * vocab * dim > cap:
        tokens //= 2
    return _loss(kind, tokens, vocab, dim, dtype, rng.choice([0.0, 0.0, 0.2, 0.5, 0.9]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + 17)


def _ids(n, vocab, g):
    """Token ids with the frequencies of text: log-uniform ranks (Zipf)."""
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)).long() - 1).clamp_(0, vocab - 1)


def _masked_count(case):
    return int(round(case["tokens"] * case["masked"]))


def _grad_shapes(case):
    """(shape, is float32 whatever the parameters' type) of a Mamba2 LM's gradients,
    in the order of its parameter dict."""
    d, v = case["dim"], case["vocab"]
    d_inner = 2 * d
    heads = max(1, d_inner // 64)
    conv = d_inner + 2 * 128
    shapes = [((v, d), False)]
    for _ in range(case["layers"]):
        shapes += [((d, d_inner + conv + heads), False), ((conv, 4), False), ((conv,), False),
                   ((heads,), True), ((heads,), True), ((heads,), True), ((d_inner,), False),
                   ((d_inner, d), False), ((d,), False)]
    return shapes + [((d,), False)]


def _flat(shapes, dt):
    """One buffer for the gradients of the parameters' type, one for the float32 ones
    (the same where the parameters are float32)."""
    sizes = {}
    for shape, f32 in shapes:
        t = torch.float32 if f32 else dt
        sizes[t] = sizes.get(t, 0) + math.prod(shape)
    return [torch.empty(n, device=DEV, dtype=t) for t, n in sizes.items()]


def _views(shapes, dt, flat):
    at = {b.dtype: 0 for b in flat}
    by = {b.dtype: b for b in flat}
    views = []
    for shape, f32 in shapes:
        t, n = torch.float32 if f32 else dt, math.prod(shape)
        views.append(by[t][at[t]:at[t] + n].view(shape))
        at[t] += n
    return views


def prepare(case, seed):
    g = _gen(seed)
    dt = _dtype(case)
    kind = case["kind"]
    if kind == "clip":
        # gradients as a data-parallel program keeps them: views of one flat buffer for
        # each type, and the like for the clipped ones
        shapes = _grad_shapes(case)
        flat = _flat(shapes, dt)
        for buf in flat:
            buf.normal_(0.0, 0.01, generator=g)
        out = _flat(shapes, dt)
        return dict(case=case, grads=_views(shapes, dt, flat), out=_views(shapes, dt, out), flat=out)
    n, v, d = case["tokens"], case["vocab"], case["dim"]
    if kind == "embed":
        w = torch.randn((v, d), generator=g, device=DEV, dtype=dt) * 0.02
        return dict(case=case, w=w, ids=_ids(n, v, g), scale=math.sqrt(d) if case["scaled"] else 1.0)
    if kind == "embed_grad":
        ids = _ids(n, v, g)
        dout = torch.randn((n, d), generator=g, device=DEV, dtype=dt) * 0.01
        return dict(case=case, ids=ids, dout=dout, scale=math.sqrt(d) if case["scaled"] else 1.0,
                    padding=0 if case["padding"] else None)
    # hidden states after the last norm, moved towards the row of the token that
    # follows by 0 to 25 in its logit: losses from near 0 to above log(vocab)
    w = torch.randn((v, d), generator=g, device=DEV) * 0.02
    targets = _ids(n, v, g)
    pull = torch.rand((n, 1), generator=g, device=DEV) * (25.0 / (0.02 ** 2 * d))
    x = torch.randn((n, d), generator=g, device=DEV) + pull * w[targets]
    drop = torch.randperm(n, generator=g, device=DEV)[:_masked_count(case)]
    targets[drop] = IGNORE
    x, w = x.to(dt), w.to(dt)
    if kind == "train":
        x.requires_grad_()
        w.requires_grad_()
    return dict(case=case, x=x, w=w, targets=targets)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _run_own(state):
    ops = _ops()
    kind = state["case"]["kind"]
    if kind == "embed":
        return ops.embedding(state["ids"], state["w"], scale=state["scale"])
    if kind == "embed_grad":
        return ops.embedding_grad(state["ids"], state["dout"], state["case"]["vocab"],
                                  scale=state["scale"], padding_idx=state["padding"])
    if kind == "clip":
        _, norm = ops.clip_grad_norm(state["grads"], state["case"]["max_norm"], out=state["out"])
        return [norm, *state["flat"]]
    if kind == "score":
        return ops.linear_cross_entropy(state["x"], state["w"], state["targets"],
                                        ignore_index=IGNORE, reduction="none")
    loss = ops.linear_cross_entropy(state["x"], state["w"], state["targets"], ignore_index=IGNORE)
    dx, dw = torch.autograd.grad(loss, (state["x"], state["w"]))
    return dict(loss=loss.detach(), dx=dx, dw=dw)


def _plain_loss(x, w, targets):
    """(per-token loss, logits - lse, targets with 0 for those left out, kept)."""
    kept = targets != IGNORE
    t = torch.where(kept, targets, torch.zeros_like(targets))
    z = x.float() @ w.float().t()
    m = z.max(dim=1, keepdim=True).values
    z -= m
    s = torch.exp(z).sum(dim=1, keepdim=True)
    logp = z - torch.log(s)
    loss = -logp.gather(1, t[:, None])[:, 0]
    return torch.where(kept, loss, torch.zeros_like(loss)), logp, t, kept


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    kind = case["kind"]
    dt = _dtype(case)
    with torch.no_grad():
        if kind == "embed":
            return (state["w"][state["ids"]].float() * state["scale"]).to(dt)
        if kind == "embed_grad":
            ids, rows = state["ids"], state["dout"].float() * state["scale"]
            if state["padding"] is not None:
                rows = torch.where((ids == state["padding"])[:, None], torch.zeros_like(rows), rows)
            out = torch.zeros((case["vocab"], case["dim"]), device=rows.device)
            return out.index_add_(0, ids, rows).to(dt)
        if kind == "clip":
            total = torch.zeros((), device=DEV, dtype=torch.float64)
            for t in state["grads"]:
                f = t.float()
                total = total + (f * f).sum(dtype=torch.float64)
            norm = total.sqrt().float()
            c = torch.clamp(case["max_norm"] / (norm + CLIP_EPS), max=1.0)
            for t, o in zip(state["grads"], state["out"]):
                o.copy_(t.float() * c)
            return [norm, *state["flat"]]
        x, w, targets = state["x"], state["w"], state["targets"]
        loss, logp, t, kept = _plain_loss(x, w, targets)
        if kind == "score":
            return loss
        count = kept.sum().clamp(min=1).float()
        gr = torch.exp(logp)
        gr.scatter_add_(1, t[:, None], torch.full_like(loss, -1.0)[:, None])
        gr *= (kept.float() / count)[:, None]
        return dict(loss=loss.sum() / count, dx=(gr @ w.float()).to(dt), dw=(gr.t() @ x.float()).to(dt))


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    es = SIZE[case["dtype"]]
    kind = case["kind"]
    if kind == "clip":
        n = b = 0
        for shape, f32 in _grad_shapes(case):
            k = math.prod(shape)
            n += k
            b += k * (4 if f32 else es)
        return {"bytes": 2 * b + 4, "flops": 3 * n}
    n, v, d = case["tokens"], case["vocab"], case["dim"]
    if kind == "embed":
        # the rows that the ids name, each of them once
        rows = min(n, v)
        return {"bytes": 8 * n + rows * d * es + n * d * es, "flops": n * d if case["scaled"] else 0}
    if kind == "embed_grad":
        return {"bytes": 8 * n + n * d * es + v * d * es, "flops": n * d}
    kept = n - _masked_count(case)
    bytes_ = 8 * n + kept * d * es + v * d * es
    if kind == "score":
        return {"bytes": bytes_ + 4 * n, "flops": 2 * kept * v * d}
    return {"bytes": bytes_ + 4 + n * d * es + v * d * es, "flops": 6 * kept * v * d}


# ---------------------------------------------------------------------------
# the results in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind == "embed":
            return torch.index_select(state["w"], 0, state["ids"]).double().mul_(state["scale"])
        if kind == "embed_grad":
            ids, dout = state["ids"], state["dout"]
            keep = torch.ones_like(ids, dtype=torch.bool) if state["padding"] is None \
                else ids != state["padding"]
            out = torch.zeros((case["vocab"], case["dim"]), device=DEV, dtype=torch.float64)
            out.index_add_(0, ids[keep], dout[keep].double())
            return out.mul_(state["scale"])
        if kind == "clip":
            sq = [torch.linalg.vector_norm(t, dtype=torch.float64) ** 2 for t in state["grads"]]
            norm = torch.stack(sq).sum().sqrt()
            c = min(1.0, case["max_norm"] / (float(norm) + CLIP_EPS))
            by = {}
            for t in state["grads"]:
                by.setdefault(t.dtype, []).append(t.reshape(-1).double().mul_(c))
            return [norm, *[torch.cat(by[b.dtype]) for b in state["flat"]]]
        x, w, targets = (state[k].detach() for k in ("x", "w", "targets"))
        n = x.shape[0]
        wd = w.double()
        kept = (targets != IGNORE).nonzero()[:, 0]
        loss = torch.zeros(n, device=DEV, dtype=torch.float64)
        dx = torch.zeros(x.shape, device=DEV, dtype=torch.float64)
        dw = torch.zeros(w.shape, device=DEV, dtype=torch.float64)
        for part in kept.split(512):
            xp = x[part].double()
            z = xp @ wd.t()
            lse = torch.logsumexp(z, dim=1)
            zt = z[torch.arange(len(part), device=DEV), targets[part]]
            loss[part] = lse - zt
            if kind == "train":
                p = torch.exp(z - lse[:, None])
                p[torch.arange(len(part), device=DEV), targets[part]] = torch.expm1(zt - lse)
                p /= max(1, len(kept))
                dx[part] = p @ wd
                dw += p.t().contiguous() @ xp
        if kind == "score":
            return loss
        return dict(loss=loss.sum() / max(1, len(kept)), dx=dx, dw=dw)
