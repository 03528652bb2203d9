"""What the vocabulary's operators once answered wrongly.  Formulas and tolerances are those of
test_gpu_vocab."""

import pytest
import torch

from gpu_util import announce
from mamba2_jax import ops
from test_gpu_vocab import DEV, DT, F, IGN, Ref, ce_inputs, gen, make_ids, u, within
from test_gpu_vocab_sizes import _bwd, _fwd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,apart", [(16, 150_000_000), (40, 60_000_000), (64, 34_100_000)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_score_rows_far_apart(n, apart, dtype):
    """The last positions of long prompts: rows of x whose offsets pass 32 bits, as those rows
    beside each other."""
    announce("rows far apart", n, apart, dtype)
    x, w, t = ce_inputs(n, 700, 128, dtype, 0.2, key=50)
    flat = torch.empty(((n - 1) * apart + 128,), device=DEV, dtype=DT[dtype])
    far = flat.as_strided((n, 128), (apart, 1))
    far.copy_(x)
    assert (n - 1) * apart * x.element_size() > 2 ** 32
    r = Ref(x, w, t, torch.ones(n, device=DEV, dtype=torch.float64))
    loss = ops.linear_cross_entropy(far, w, t, reduction="none")
    within(loss, r.loss, r.loss_tol, "loss")
    assert not bool(loss[t == IGN].any())


@pytest.mark.parametrize("n", [1, 16, 17, 64])
@pytest.mark.parametrize("dim", [64, 192, 256, 320, 448, 576, 832, 2560])
def test_score_last_step_in_each_slot(n, dim):
    """Few tokens: the wavefronts of a tile put their sums together in LDS that no operand lies in,
    whichever slot of the ring (of four up to 16 tokens, of three beyond) the last K step
    is in.  16 runs of more tiles than the card has CUs, equal to the bit."""
    announce("last step in each slot", n, dim)
    x, w, t = ce_inputs(n, 128 * 300, dim, "bf16", key=51)
    r = Ref(x, w, t, torch.ones(n, device=DEV, dtype=torch.float64))
    loss = ops.linear_cross_entropy(x, w, t, reduction="none")
    within(loss, r.loss, r.loss_tol, "loss")
    for _ in range(15):
        assert torch.equal(ops.linear_cross_entropy(x, w, t, reduction="none"), loss)


def dw_tolerance(x, w, t, up):
    """(dw, its tolerance) of test_gpu_vocab's Ref, in which G at the target is not rounded to
    bfloat16: what that would take from it is added in float32, off by the roundings of its products
    and sums."""
    r = Ref(x, w, t, up)
    kept = t != IGN
    X, tt = x.double()[kept], t[kept]
    z = X @ w.double().t()
    G = up[kept] * torch.expm1(z.gather(1, tt[:, None])[:, 0] - torch.logsumexp(z, 1))
    half = u(torch.bfloat16)
    at = torch.zeros_like(r.dw).index_add_(0, tt, G.abs()[:, None] * X.abs())
    count = torch.bincount(tt, minlength=len(w)).double()[:, None]
    # what an unmended dw would be
    lost = torch.zeros_like(r.dw).index_add_(0, tt, (G.float().bfloat16().double() - G)[:, None] * X)
    return r.dw, r.dw_tol - half * at + half * (count + 8) * F * at, r.dw + lost


# tokens, kept, vocabulary, width, how the targets fall, one gradient of all losses or one of each
DW = [(500, 60, 5000, 136, "any", "each"), (600, 60, 5000, 136, "any", "each"), (40, 40, 3000, 64, "any", "each"),
      (64, 64, 3000, 700, "same", "each"), (65, 65, 3000, 72, "same", "each"), (700, 700, 5000, 128, "zipf", "each"),
      (700, 600, 20000, 264, "zipf", "one"), (1500, 1500, 900, 64, "same", "each"),
      (2100, 1300, 4000, 96, "same", "one"), (3000, 2500, 5000, 1001, "zipf", "each"),
      (5000, 4400, 60011, 72, "zipf", "each")]


@pytest.mark.parametrize("n,kept,vocab,dim,how,up", DW)
def test_dw_gets_back_what_the_target_lost(n, kept, vocab, dim, how, up):
    """bfloat16: dw of any number of tokens, of targets that many share, over several pieces of
    the vocabulary (the last case), whatever share of the tokens is kept."""
    announce("dw's target", n, kept, vocab, dim, how, up)
    g = gen(52, n, kept, vocab)
    w = (torch.randn((vocab, dim), generator=g, device=DEV) / dim ** 0.5).to(torch.bfloat16)
    x = torch.randn((n, dim), generator=g, device=DEV).to(torch.bfloat16)
    t = make_ids(n, vocab, how, g)
    if vocab == 60011:
        t[::7] = vocab - 1 - torch.arange(len(t[::7]), device=DEV) % 5
    t[torch.randperm(n, generator=g, device=DEV)[:n - kept]] = IGN
    if up == "one":
        ups = torch.full((n,), 0.7, device=DEV)
        arg, reduction = torch.tensor(0.7, device=DEV), "sum"
    else:
        ups = arg = torch.rand(n, generator=g, device=DEV) + 0.5
        reduction = "none"
    wg = w.clone().requires_grad_()
    loss = ops.linear_cross_entropy(x, wg, t, reduction=reduction)
    dw, = torch.autograd.grad(loss, wg, arg, retain_graph=True)
    want, tol, unmended = dw_tolerance(x, w, t, ups.double())
    within(dw, want, tol, "dw")
    assert torch.equal(torch.autograd.grad(loss, wg, arg)[0], dw)
    if up == "each":
        assert bool(((unmended.to(torch.bfloat16).double() - want).abs() > tol).any()), "would not be noticed"


def far_below(n, dtype):
    """Inputs whose targets' logits are -10000 and the others of the order of ten (exact in bfloat16)."""
    g = gen(53, n)
    w = torch.randint(-8, 9, (300, 64), generator=g, device=DEV) / 16.0
    x = torch.randint(-8, 9, (n, 64), generator=g, device=DEV) / 4.0
    w[:, 0], x[:, 0] = 0.0, 100.0
    t = torch.randint(0, 40, (n,), generator=g, device=DEV)
    w[:40] = 0.0
    w[:40, 0] = -100.0
    return x.to(DT[dtype]), w.to(DT[dtype]), t


@pytest.mark.parametrize("n", [9, 40, 300])
@pytest.mark.parametrize("saved", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_lse_of_targets_far_below(n, saved, dtype):
    """lse does not depend on how far below the others the target lies.  The logits are exact (multiples
    of 1 / 64 below 1024 in size, as are all their partial sums), so its error is a rounding
    each for the exponentials' arguments, the maximum and the result, and those of a sum of 300."""
    announce("lse far below", n, saved, dtype)
    x, w, t = far_below(n, dtype)
    loss, lse, total, buf = _fwd(x, w, t, saved=saved)
    z = x.double() @ w.double().t()
    want = torch.logsumexp(z, 1)
    top = z[:, 40:].abs().max()
    tol = F * (100 + 8 * top)
    within(lse, want, tol.expand(n), "lse")
    assert tol < 1e4 * F / 2, "would not be noticed"
    # the softmax in float32's gradient: dw of the rows that are nobody's target
    if dtype == "f32":
        _, dw = _bwd(x, w, t, loss, lse, buf, mean=0)
        p = 1.5 * torch.softmax(z, 1)[:, 40:]
        ref, mag = p.t() @ x.double(), p.t() @ x.abs().double()
        e = 1.05 * (2 * tol + 8 * F * (top + 8)) + (6 * (n / 4 + 32) + 16) * F
        within(dw[40:], ref, e * mag + F * ref.abs() + 1e-42, "dw")


@pytest.mark.parametrize("n", [5, 40, 300])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("where", ["target", "other"])
@pytest.mark.parametrize("sign", [1, -1])
def test_infinite_logits(n, dtype, where, sign):
    """A logit of +inf has no softmax: NaN, as exp(z - max) gives it.  One of -inf has none of it: loss inf
    if it is the target's, and gradients that are finite all the same."""
    announce("infinite logits", n, dtype, where, sign)
    x, w, t = ce_inputs(n, 300, 64, dtype, key=54)
    t = torch.arange(n, device=DEV) % 299
    t[1] = 299
    x[:, 0], w[:, 0] = 0.0, 0.0
    row = 1 if where == "target" else 3                 # its logit of weight row 299 is infinite
    x[row, 0], w[299, 0] = sign * 2.0 ** 100, 2.0 ** 100
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    saved = ops.linear_cross_entropy(xg, wg, t, reduction="none")
    alone = ops.linear_cross_entropy(x, w, t, reduction="none")
    dx, dw = torch.autograd.grad(saved.sum(), (xg, wg))
    z = x.double() @ w.double().t()
    z[row, 299] = sign * float("inf")
    p = torch.exp(z - z.max(1, keepdim=True).values)
    p /= p.sum(1, keepdim=True)
    rest = torch.arange(n, device=DEV) != row
    for loss in (saved.detach(), alone):
        if sign > 0:
            assert bool(loss[row].isnan())
        elif where == "target":
            assert float(loss[row]) == float("inf")
        assert bool(loss[rest].isfinite().all())
        assert bool(ops.linear_cross_entropy(x, w, t).isnan()) == (sign > 0)
    assert bool(dx[rest].isfinite().all())
    if sign > 0:
        assert bool(dx[row].isnan().all()) and bool(dw.isnan().all())
        return
    G = p - torch.nn.functional.one_hot(t, 300)
    # G's rounding and the result's; the logits' error, 6 (64 / 4 + 16) F of at most 20, twice
    lim = 2.0 ** -11 + (2.0 ** -7 if dtype == "bf16" else 0.0)
    want = G @ w.double()
    assert bool(((dx.double() - want).abs() <= lim * (G.abs() @ w.abs().double()) + 1e-30).all())
    want = G.t().contiguous() @ x.double()
    assert bool(((dw.double() - want).abs() <= lim * (G.abs().t().contiguous() @ x.abs().double()) + 1e-30).all())


@pytest.mark.parametrize("n,vocab", [(512 * 2048, 3000), (512 * 2048 + 1, 300000), (1025 * 2048 - 7, 70000),
                                     (5_000_011, 2 ** 26)])
def test_embedding_grad_of_many_entries(n, vocab):
    """More tiles than the sort has workgroups.  Whole numbers, whose sums are exact."""
    announce("many entries", n, vocab)
    g = gen(55, n)
    ids = make_ids(n, vocab, "any" if n & 1 else "zipf", g)
    ids[n // 3], ids[n // 2] = vocab, -1
    grad = torch.randint(-3, 4, (n, 2), generator=g, device=DEV).float()
    want = torch.zeros(vocab + 1, 2, dtype=torch.float64, device=DEV)
    want.index_add_(0, torch.where((ids < 0) | (ids > vocab), vocab, ids), grad.double())
    assert torch.equal(ops.embedding_grad(ids, grad, vocab).double(), want[:vocab])
    # the order of a token's entries is theirs: (2^24 + 1) - 2^24 is 0 in float32 (four entries a token:
    # none is summed in two parts, which begin at multiples of four)
    k = n // 4
    ids = torch.arange(4 * k, device=DEV) % k
    vals = torch.tensor([2.0 ** 24, 1.0, -(2.0 ** 24), 0.0], device=DEV)[torch.arange(4 * k, device=DEV) // k]
    assert not bool(ops.embedding_grad(ids, vals[:, None], k).any())
