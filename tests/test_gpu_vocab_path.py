"""The vocabulary's operators where they are used together: a bigram model's training steps
(examples/bigram_lm.py) and the scoring of a Mamba2 LM."""

import math
import os
import sys

import pytest
import torch

from gpu_util import announce
from mamba2_jax.models import Mamba2Config, Mamba2LMHeadModel, init_params

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import bigram_lm  # noqa: E402

pytestmark = pytest.mark.gpu

CFG = Mamba2Config(d_model=128, n_layer=3, vocab_size=300, d_state=64, headdim=64, ngroups=1, chunk_size=64)
F, UB = 2.0 ** -24, 2.0 ** -9          # half steps of float32 and (twice) bfloat16


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_bigram_learns(dtype):
    """The loss leaves log(vocab) for the entropy of the text, and two runs are equal bit for bit."""
    announce("bigram", dtype)
    kw = dict(vocab=500, dim=64, tokens=2000, steps=60, dtype=dtype)
    a, b = bigram_lm.train(**kw), bigram_lm.train(**kw)
    assert torch.equal(a, b)
    print(f"  {a[0]:.3f} -> {a[-1]:.3f}", flush=True)
    assert a[0] > 0.9 * math.log(500) and a[-1] < 0.7 * math.log(500)


def test_bigram_step_against_autograd():
    """One step of float32 against torch's own operators in 64 bits."""
    announce("bigram step")
    g = torch.Generator(device="cuda").manual_seed(3)
    e, w = (torch.randn((70, 24), generator=g, device="cuda") for _ in range(2))
    ids, t = (torch.randint(0, 70, (90,), generator=g, device="cuda") for _ in range(2))
    p = [v.double().requires_grad_() for v in (e, w)]
    z = p[0][ids] @ p[1].t()
    loss = (torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0]).mean()
    grads = torch.autograd.grad(loss, p)
    norm = torch.sqrt(sum((v * v).sum() for v in grads))
    c = min(1.0, 0.5 / (float(norm) + 1e-6))
    got = [v.clone().requires_grad_() for v in (e, w)]
    l2, n2 = bigram_lm.step(*got, ids, t, 0.25, 0.5)
    # the logits are off by 6 (24 / 4 + 16) F of their products' absolute sums, which the
    # softmax passes on as often as there are terms in what follows
    dz = 6 * 22 * F * float((e[ids].abs().double() @ w.abs().double().t()).max())
    assert abs(float(l2) - float(loss)) <= 2 * dz + 60 * F * float(z.abs().max())
    rel = 4 * dz + 300 * F
    assert abs(float(n2) - float(norm)) <= rel * float(norm) * 10
    for q, v, gr in zip(got, (e, w), grads):
        want = v.double() - 0.25 * c * gr
        mag = gr.abs().max()
        assert bool(((q.double() - want).abs() <= 0.25 * 20 * rel * mag + 2 * F * v.abs()).all())


def _cast(v, dtype):
    if isinstance(v, dict):
        return {k: _cast(x, dtype) for k, x in v.items()}
    if isinstance(v, list):
        return [_cast(x, dtype) for x in v]
    return v.to(dtype) if v is not None and v.dtype == torch.bfloat16 else v


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual32", [True, False])
def test_lm_score(dtype, residual32):
    """score() against the cross entropy in 64 bits of the logits that the model answers with.
    Those multiply the float32 final norm, score() the norm rounded to the head's dtype: a logit
    differs by UB of the sum of its products' absolute values at most (bfloat16), and by the
    float32 sums' errors."""
    announce("lm score", dtype, residual32)
    cfg = Mamba2Config(**{**CFG.__dict__, "residual_in_fp32": residual32})
    params = _cast(init_params(cfg, seed=2), dtype)
    model = Mamba2LMHeadModel(cfg)
    g = torch.Generator(device="cuda").manual_seed(4)
    ids = torch.randint(0, cfg.vocab_size, (2, 130), generator=g, device="cuda")
    z = model(params, ids).double()
    w = params["lm_head_weight"].double()
    targets = torch.randint(0, cfg.vocab_size, ids.shape, generator=g, device="cuda")
    targets[0, :40] = -100
    for t in (targets, None):
        tt = targets if t is not None else torch.cat([ids[:, 1:], torch.full_like(ids[:, :1], -100)], 1)
        kept = tt != -100
        lse = torch.logsumexp(z, -1)
        want = torch.where(kept, lse - z.gather(-1, tt.clamp(min=0)[..., None])[..., 0], torch.zeros_like(lse))
        got = model.score(params, ids, t)
        assert got.dtype == torch.float32 and got.shape == ids.shape
        # |xn| <= sqrt(d_model) per row (a norm with weight one)
        products = math.sqrt(cfg.d_model) * w.norm(dim=1).max()
        tol = 2 * products * ((UB if dtype == torch.bfloat16 else 0) + 600 * F) + 200 * F
        err = (got.double() - want).abs().max()
        print(f"  error {float(err):.2e}, tolerance {float(tol):.2e}", flush=True)
        assert bool(err <= tol)
        assert not bool(got[~kept].any())
        mean = model.score(params, ids, t, reduction="mean")
        assert abs(float(mean) - float(got.double().sum() / kept.sum())) <= 4 * F * float(mean)
    # a head of its own that learns
    head = params["lm_head_weight"].detach().clone().requires_grad_()
    loss = model.score({**params, "lm_head_weight": head}, ids, targets, reduction="mean")
    (gh,) = torch.autograd.grad(loss, head)
    assert gh.shape == head.shape and bool(gh.isfinite().all()) and float(gh.abs().max()) > 0


def test_lm_score_refuses():
    params = init_params(CFG, seed=2)
    ids = torch.zeros((1, 8), dtype=torch.long, device="cuda")
    with pytest.raises(AssertionError):
        Mamba2LMHeadModel(CFG).score(params, ids, ids[:, :4])
    with pytest.raises(AssertionError):
        Mamba2LMHeadModel(CFG).score(params, ids, reduction="max")
