"""Train a bigram language model, p(next | token) = softmax(head @ embedding[token]), with the
vocabulary's operators: the lookup and its gradient by sorted tokens, the loss of the linear head
without its logits, and clipping by the global gradient norm.  Such a model is the smallest
draft model that a decoder can be given, and everything around a Mamba2 LM's layers in a
training step.

    python examples/bigram_lm.py [--vocab 8192] [--dim 256] [--tokens 8192] [--steps 100]

The text is synthetic: each token is followed by one fixed successor four times out of five,
by any token otherwise, so the loss falls from log(vocab) towards the entropy of that, printed first.
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "mamba2-jax-pallas_amd"))

from mamba2_jax import ops  # noqa: E402

SURE = 0.8


def batch(successor, tokens, generator):
    """-> (tokens, their successors), both (tokens,)."""
    vocab, dev = successor.numel(), successor.device
    ids = torch.randint(0, vocab, (tokens,), generator=generator, device=dev)
    anything = torch.randint(0, vocab, (tokens,), generator=generator, device=dev)
    sure = torch.rand(tokens, generator=generator, device=dev) < SURE
    return ids, torch.where(sure, successor[ids], anything)


def step(embedding, head, ids, targets, lr, max_norm):
    """One step of gradient descent on embedding and head, in place -> (loss, gradient norm)."""
    with torch.enable_grad():
        hidden = ops.embedding(ids, embedding)
        loss = ops.linear_cross_entropy(hidden, head, targets)
    grads = torch.autograd.grad(loss, (embedding, head))
    grads, norm = ops.clip_grad_norm(grads, max_norm, out=grads)
    with torch.no_grad():
        for p, g in zip((embedding, head), grads):
            p.sub_(g, alpha=lr)
    return loss.detach(), norm


def train(vocab=8192, dim=256, tokens=8192, steps=100, lr=None, max_norm=1.0, dtype=torch.float32,
          seed=0, report=None):
    """-> the losses of all steps, (steps,) on the CPU."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    successor = torch.randperm(vocab, generator=g, device="cuda")
    embedding, head = (torch.randn((vocab, dim), generator=g, device="cuda").mul_(dim ** -0.25)
                       .to(dtype).requires_grad_() for _ in range(2))
    # a visit of a token moves its successor's logit by about a quarter
    lr = tokens / dim ** 0.5 / 4 if lr is None else lr
    losses = []
    for i in range(steps):
        ids, targets = batch(successor, tokens, g)
        loss, norm = step(embedding, head, ids, targets, lr, max_norm)
        losses.append(loss)
        if report and (i % 10 == 0 or i == steps - 1):
            report(f"step {i:4d}  loss {float(loss):7.4f}  gradient norm {float(norm):.4f}")
    return torch.stack(losses).cpu()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("vocab", 8192), ("dim", 256), ("tokens", 8192), ("steps", 100)):
        ap.add_argument(f"--{name}", type=int, default=default)
    ap.add_argument("--bf16", action="store_true")
    a = ap.parse_args(argv)
    floor = -SURE * math.log(SURE + (1 - SURE) / a.vocab) \
        - (1 - SURE) * math.log((1 - SURE) / a.vocab)
    print(f"log(vocab) {math.log(a.vocab):.4f}, entropy of the text {floor:.4f}")
    train(a.vocab, a.dim, a.tokens, a.steps, dtype=torch.bfloat16 if a.bf16 else torch.float32,
          report=print)


if __name__ == "__main__":
    main()
