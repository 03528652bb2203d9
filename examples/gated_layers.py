"""A small language model of residual layers that can be trained: embedding, then in each layer the
gated linear recurrence over time and the gated feed-forward product over the channels, then the head's loss
without its logits and the clipping of the gradients.  One layer:

    x, r, i = u W_in           (one projection; its thirds are read in place)
    u = u + recurrence(x, r, i, -exp(A_log)) W_out
    u = u + gated_linear(u, W_up) W_down

    python examples/gated_layers.py [--vocab 512] [--dim 128] [--layers 2] [--seqlen 512] [--steps 20]
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if os.path.join(ROOT, "mamba2-jax-pallas_amd") not in sys.path:
    sys.path.insert(0, os.path.join(ROOT, "mamba2-jax-pallas_amd"))

from mamba2_jax import ops  # noqa: E402


def init(vocab, dim, hidden, layers, dtype=torch.bfloat16, seed=0):
    """Random parameters, a dict of lists of tensors."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def w(*shape, scale):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype).requires_grad_()
    blocks = []
    for _ in range(layers):
        A_log = torch.empty(dim, device="cuda").uniform_(math.log(1e-3), math.log(0.3), generator=g)
        blocks.append({"w_in": w(dim, 3 * dim, scale=dim ** -0.5), "A_log": A_log.requires_grad_(),
                       "w_out": w(dim, dim, scale=0.5 * dim ** -0.5), "w_up": w(2 * hidden, dim, scale=dim ** -0.5),
                       "w_down": w(hidden, dim, scale=0.5 * hidden ** -0.5)})
    return {"embedding": w(vocab, dim, scale=1.0), "blocks": blocks, "head": w(vocab, dim, scale=dim ** -0.5)}


def leaves(params):
    return [params["embedding"], *(t for b in params["blocks"] for t in b.values()), params["head"]]


def layer(u, b, states=None, seq_idx=None):
    """u (batch, seqlen, dim) -> (u behind the layer, final states)"""
    x, r, i = (u @ b["w_in"]).chunk(3, dim=-1)
    h, last = ops.gated_linear_recurrence(x, r, i, -torch.exp(b["A_log"]), initial_states=states, seq_idx=seq_idx,
                                          return_final_states=True)
    u = u + h @ b["w_out"]
    return u + ops.gated_linear(u, b["w_up"]) @ b["w_down"], last


def layer_step(u, b, state):
    """One token, under torch.no_grad(): u (batch, dim), state updated in place -> u behind the layer"""
    x, r, i = (u @ b["w_in"]).chunk(3, dim=-1)
    _, h = ops.gated_linear_recurrence_update(state, x, r, i, -torch.exp(b["A_log"]), inplace=True)
    u = u + h @ b["w_out"]
    return u + ops.gated_linear(u, b["w_up"]) @ b["w_down"]


def loss_of(params, ids, targets, seq_idx=None):
    u = ops.embedding(ids, params["embedding"])
    for b in params["blocks"]:
        u, _ = layer(u, b, seq_idx=seq_idx)
    return ops.linear_cross_entropy(u, params["head"], targets)


def step(params, ids, targets, lr=0.1, max_norm=1.0, seq_idx=None):
    """One training step, parameters updated in place -> (loss, gradient norm)"""
    ps = leaves(params)
    loss = loss_of(params, ids, targets, seq_idx)
    grads = list(torch.autograd.grad(loss, ps))
    grads, norm = ops.clip_grad_norm(grads, max_norm, out=grads)
    with torch.no_grad():
        for p, g in zip(ps, grads):
            p.sub_(lr * g)
    return loss.detach(), norm


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__)
    for name, value in (("vocab", 512), ("dim", 128), ("layers", 2), ("seqlen", 512), ("steps", 20)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args(argv)
    params = init(a.vocab, a.dim, 2 * a.dim, a.layers)
    g = torch.Generator(device="cuda").manual_seed(1)
    for k in range(a.steps):
        start = torch.randint(0, a.vocab, (4, 1), generator=g, device="cuda")
        ids = (start + 7 * torch.arange(a.seqlen + 1, device="cuda")) % a.vocab
        loss, norm = step(params, ids[:, :-1], ids[:, 1:])
        print(f"step {k}: loss {float(loss):.3f}, gradient norm {float(norm):.3f}", flush=True)


if __name__ == "__main__":
    main()
