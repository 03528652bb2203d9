"""The vocabulary's operators (linear_cross_entropy, embedding, embedding_grad,
clip_grad_norm) against plain 64-bit formulas.

Tolerances are per element and derived from the arithmetic, u(T) being half a step
(torch.finfo(T).eps / 2) and F = 2^-24:
* a stored result is off by u(T) |ref|;
* a float32 sum of n terms by at most n F sum |term|;
* a matrix product over K by (K / 4 + 16) F sum |a b| (one instruction adds 32 products in at
  most eight roundings); float32 operands run six such sums and leave out 4 F;
* the loss by the logits' error twice, F for each of the sums' roundings and of the
  values that enter the difference;
* G by its relative rounding (u(bf16), or 4 F for float32 operands) and the errors of
  logit and lse that enter the exponential.
"""

import math

import numpy as np
import pytest
import torch

from gpu_util import announce
from mamba2_jax import ops

pytestmark = pytest.mark.gpu

F = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
DEV = "cuda"


def u(dtype):
    return torch.finfo(dtype).eps / 2


def gen(*key):
    return torch.Generator(device=DEV).manual_seed(hash(key) % (2 ** 31))


def within(got, want, tol, what):
    got = got.detach().double()
    bad = ~((got - want).abs() <= tol)
    both_nan = got.isnan() & want.isnan()
    bad &= ~both_nan
    worst = float(((got - want).abs() / tol.clamp_min(1e-300)).nan_to_num(0.0).max()) if got.numel() else 0.0
    print(f"  {what}: worst error / tolerance {worst:.3f}", flush=True)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the tolerance"


# ---------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------
LOOKUPS = [(1, 7, 8), (16, 50288, 2560), (5, 3, 1), (33, 1000, 1001), (700, 333, 130), (4099, 50277, 768),
           (2, 1, 4096), (64, 97, 1028)]


@pytest.mark.parametrize("n,vocab,dim", LOOKUPS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [1.0, 7.7])
def test_embedding(n, vocab, dim, dtype, scale):
    announce("embedding", n, vocab, dim, dtype, scale)
    g = gen(1, n, vocab, dim)
    w = torch.randn((vocab, dim), generator=g, device=DEV).to(DT[dtype])
    ids = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    out = ops.embedding(ids, w, scale=scale)
    ref = w[ids].double() * scale
    if scale == 1.0:
        assert torch.equal(out, w[ids])
    else:
        within(out, ref, ref.abs() * (u(DT[dtype]) + 2 * F) + 1e-45, "rows")
    assert torch.equal(out, ops.embedding(ids.int().view(n, 1), w, scale=scale).view(n, dim))


def test_embedding_views_and_bad_ids():
    announce("embedding views")
    g = gen(2)
    base = torch.randn((40, 300), generator=g, device=DEV)
    for w in (base[:, 4:204], base[:, 3:104], base.to(torch.bfloat16)[::2, 1:130], base.t()):
        ids = torch.randint(0, w.shape[0], (3, 5), generator=g, device=DEV)
        assert torch.equal(ops.embedding(ids, w), w[ids])
    w = base[:, :64]
    ids = torch.tensor([0, -1, 40, 39, 2 ** 40], device=DEV)
    out = ops.embedding(ids, w)
    assert torch.equal(out[[0, 3]], w[[0, 39]])
    assert bool(out[[1, 2, 4]].isnan().all())
    assert ops.embedding(ids[:0], w).shape == (0, 64)


def grad_ref(ids, grad, vocab, scale, padding):
    """(rows, sums of absolute values, entries) in 64 bits."""
    keep = (ids >= 0) & (ids < vocab)
    if padding is not None:
        keep &= ids != padding
    i, d = ids[keep].long(), grad[keep].double() * scale
    out = torch.zeros((vocab, grad.shape[-1]), dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(out)
    out.index_add_(0, i, d)
    mag.index_add_(0, i, d.abs())
    return out, mag, torch.bincount(i, minlength=vocab).double()[:, None]


# (n, vocab, dim, how the ids fall)
GRADS = [(0, 9, 16, "any"), (1, 1, 1, "any"), (1, 50288, 64, "any"), (7, 5, 24, "any"), (64, 64, 8, "same"),
         (4095, 1000, 33, "zipf"), (4096, 70001, 8, "zipf"), (4097, 70001, 8, "zipf"), (5000, 3, 40, "any"),
         (6001, 100, 72, "same"), (16384, 50277, 128, "zipf"), (20000, 300000, 16, "any"),
         (2047, 512, 4100, "zipf"), (9000, 511, 5, "any"), (333, 32003, 1001, "zipf")]


def make_ids(n, vocab, how, g):
    if how == "same":
        return torch.full((n,), vocab // 2, device=DEV, dtype=torch.long)
    if how == "any":
        return torch.randint(0, vocab, (n,), generator=g, device=DEV)
    r = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    return (torch.exp(r * math.log(vocab + 1)).long() - 1).clamp_(0, vocab - 1)


@pytest.mark.parametrize("n,vocab,dim,how", GRADS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_embedding_grad(n, vocab, dim, how, dtype):
    announce("embedding_grad", n, vocab, dim, how, dtype)
    g = gen(3, n, vocab, dim)
    ids = make_ids(n, vocab, how, g)
    grad = torch.randn((n, dim), generator=g, device=DEV).to(DT[dtype])
    padding = int(ids[0]) if n > 3 and how == "zipf" else None
    for scale in (1.0, 3.3):
        ref, mag, cnt = grad_ref(ids, grad, vocab, scale, padding)
        out = ops.embedding_grad(ids, grad, vocab, scale=scale, padding_idx=padding)
        assert out.dtype == grad.dtype
        within(out, ref, u(out.dtype) * ref.abs() + (cnt + 3) * F * mag * 1.01 + 1e-45 * (cnt > 0), "rows")
        assert torch.equal(out, ops.embedding_grad(ids.int(), grad, vocab, scale=scale, padding_idx=padding))


@pytest.mark.parametrize("gdt,odt", [("bf16", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("n,vocab,dim", [(300, 77, 40), (5001, 1234, 72), (100, 50, 9)])
def test_embedding_grad_into(gdt, odt, n, vocab, dim):
    """out=: added to in place, the rows that no id names untouched; dtype=."""
    announce("embedding_grad into", gdt, odt, n, vocab, dim)
    g = gen(4, n, dim)
    ids = make_ids(n, vocab, "zipf", g)
    ids[5] = vocab                                  # takes no part
    ids[6] = -7
    grad = torch.randn((n, dim), generator=g, device=DEV).to(DT[gdt])
    ref, mag, cnt = grad_ref(ids, grad, vocab, 0.5, None)
    out = ops.embedding_grad(ids, grad, vocab, scale=0.5, dtype=DT[odt])
    assert out.dtype == DT[odt]
    tol = u(out.dtype) * ref.abs() + (cnt + 3) * F * mag * 1.01
    within(out, ref, tol, "rows")
    wide = torch.randn((vocab, dim + 8), generator=g, device=DEV).to(DT[odt])
    for view in (wide[:, :dim], wide[:, 3:3 + dim]):
        keep, before, version = wide.clone(), view.clone(), view._version
        got = ops.embedding_grad(ids, grad, vocab, scale=0.5, out=view)
        assert got is view and view._version > version
        want = before.double() + ref
        within(view, want, u(out.dtype) * want.abs() + F * before.double().abs() + (cnt + 4) * F * mag * 1.01,
               "added")
        unnamed = cnt[:, 0] == 0
        assert torch.equal(view[unnamed], before[unnamed])
        view.copy_(keep[:, :dim] if view.data_ptr() == wide.data_ptr() else keep[:, 3:3 + dim])
        assert torch.equal(wide, keep)              # nothing beside the view changed


def test_embedding_autograd():
    announce("embedding autograd")
    g = gen(5)
    w = torch.randn((50, 24), generator=g, device=DEV, dtype=torch.float32).requires_grad_()
    ids = torch.randint(0, 50, (4, 9), generator=g, device=DEV)
    up = torch.randn((4, 9, 24), generator=g, device=DEV)
    (dw,) = torch.autograd.grad(ops.embedding(ids, w, scale=2.0, padding_idx=-1), w, up)
    ref, mag, cnt = grad_ref(ids.view(-1), up.view(-1, 24), 50, 2.0, 49)
    within(dw, ref, (cnt + 4) * F * mag, "dw")
    # a gradient that autograd expands (no strides of its own)
    (dw,) = torch.autograd.grad(ops.embedding(ids, w).sum(), w)
    cnt = torch.bincount(ids.view(-1), minlength=50).float()[:, None]
    assert torch.equal(dw, cnt.expand(50, 24))
    assert not ops.embedding(ids, w.detach()).requires_grad


# ---------------------------------------------------------------------------
# linear_cross_entropy
# ---------------------------------------------------------------------------
IGN = -100


def ce_inputs(n, vocab, dim, dtype, masked=0.0, key=0, std=1.0):
    g = gen(6, n, vocab, dim, key)
    w = torch.randn((vocab, dim), generator=g, device=DEV) / math.sqrt(dim)
    t = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    x = torch.randn((n, dim), generator=g, device=DEV) * std
    x += torch.rand((n, 1), generator=g, device=DEV) * 12.0 * w[t]
    if masked:
        t[torch.rand(n, generator=g, device=DEV) < masked] = IGN
    return x.to(DT[dtype]), w.to(DT[dtype]), t


class Ref:
    """The formula in 64 bits, with the tolerances of the module's docstring."""

    def __init__(self, x, w, t, up):
        """up: the upstream gradient of each position's loss (n,), 64 bits."""
        f32 = x.dtype == torch.float32
        n, dim = x.shape
        vocab = w.shape[0]
        X, W = x.detach().double(), w.detach().double()
        kept = t != IGN
        X = torch.where(kept[:, None], X, torch.zeros_like(X))
        tt = torch.where(kept, t, torch.zeros_like(t)).long()
        mm = (6 if f32 else 1) * (dim / 4 + 16) * F + (4 * F if f32 else 0)
        z = X @ W.t()
        dz = (mm * (X.abs() @ W.abs().t())).max(dim=1).values
        lse = torch.logsumexp(z, 1)
        zt = z.gather(1, tt[:, None])[:, 0]
        m = z.max(1).values
        zero = torch.zeros_like(lse)
        self.loss = torch.where(kept, lse - zt, zero)
        dl = 2 * dz + F * (130 + vocab / 2000 + 4 * (m.abs() + zt.abs() + (lse - m) + 4))
        self.loss_tol = torch.where(kept, dl, zero)
        up = torch.where(kept, up, zero)
        p = torch.exp(z - lse[:, None])
        G = p.clone()
        G.scatter_(1, tt[:, None], torch.expm1(zt - lse)[:, None])
        G *= up[:, None]
        # the exponential's argument: the logit, lse (the loss's error at most) and their
        # difference's own roundings
        e = dz + dl + F * (4 * (m.abs() + lse.abs()) + 8)
        dG = G.abs() * (4 * F if f32 else u(torch.bfloat16)) + 1.05 * up.abs()[:, None] * p * e[:, None]
        add = (6 if f32 else 1) * F

        def out(a, da, b, k, dt):
            ref = a @ b
            tol = (da + (add * (k / 4 + 32) + 4 * F) * (a.abs() + da)) @ b.abs()
            return ref, 1.01 * tol + u(dt) * ref.abs() + 1e-42
        self.dx, self.dx_tol = out(G, dG, W, vocab, x.dtype)
        self.dw, self.dw_tol = out(G.t().contiguous(), dG.t().contiguous(), X, n, w.dtype)


def ce_check(x, w, t, reduction, up=None):
    n = x.shape[0]
    x = x.detach().requires_grad_()
    w = w.detach().requires_grad_()
    kept = int((t != IGN).sum())
    loss = ops.linear_cross_entropy(x, w, t, reduction=reduction)
    assert loss.dtype == torch.float32
    if reduction == "none":
        up = torch.ones(n, device=DEV) if up is None else up
        dx, dw = torch.autograd.grad(loss, (x, w), up)
        r = Ref(x, w, t, up.double())
        within(loss, r.loss, r.loss_tol, "loss")
    else:
        up = torch.tensor(1.0 if up is None else up, device=DEV)
        dx, dw = torch.autograd.grad(loss, (x, w), up)
        d = max(kept, 1) if reduction == "mean" else 1
        r = Ref(x, w, t, (up.double() / d).expand(n))
        within(loss, r.loss.sum() / d, r.loss_tol.sum() / d + 2 * F * r.loss.sum() / d, "loss")
    assert dx.dtype == x.dtype and dw.dtype == w.dtype and dx.shape == x.shape and dw.shape == w.shape
    within(dx, r.dx, r.dx_tol, "dx")
    within(dw, r.dw, r.dw_tol, "dw")
    return loss, dx, dw


# sizes on either side of every tile (16 / 64 / 256 tokens, 128 / 256 rows of the
# vocabulary, K steps of 64, 8 elements of a row)
CE = [(1, 1, 1), (1, 50288, 768), (2, 130, 64), (15, 257, 72), (16, 128, 8), (17, 129, 65), (63, 1000, 200),
      (64, 255, 128), (65, 256, 127), (129, 511, 264), (255, 513, 40), (256, 300, 1001), (257, 4000, 96),
      (333, 32003, 136), (700, 700, 320), (1025, 2050, 520)]


@pytest.mark.parametrize("n,vocab,dim", CE)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_linear_cross_entropy(n, vocab, dim, dtype):
    announce("linear_cross_entropy", n, vocab, dim, dtype)
    masked = [0.0, 0.3, 0.9][(n + vocab + dim) % 3]
    x, w, t = ce_inputs(n, vocab, dim, dtype, masked)
    ce_check(x, w, t, ["mean", "sum", "none"][(n + dim) % 3])


@pytest.mark.parametrize("n", [5, 40, 300])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_ce_reductions_and_upstream(n, dtype):
    announce("ce reductions", n, dtype)
    x, w, t = ce_inputs(n, 500, 96, dtype, 0.4)
    ce_check(x, w, t, "mean", up=-3.0)
    ce_check(x, w, t.int(), "sum", up=0.25)
    g = gen(7, n)
    ce_check(x, w, t, "none", up=torch.randn(n, generator=g, device=DEV))
    ce_check(x, w, t, "none", up=torch.randn(2 * n, generator=g, device=DEV)[::2])
    # batches and an upstream gradient without strides
    xb, tb = x.view(1, n, 96).requires_grad_(), t.view(1, n)
    loss = ops.linear_cross_entropy(xb, w, tb, reduction="none")
    assert loss.shape == (1, n)
    a = torch.autograd.grad(loss.sum(), xb)[0]
    b = torch.autograd.grad(ops.linear_cross_entropy(xb, w, tb, reduction="sum"), xb)[0]
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [9, 400])
def test_ce_rows_left_out(n, dtype):
    """What stands in a row that is left out reaches nothing, whatever it is; all rows left out
    give zeros."""
    announce("ce masked rows", n, dtype)
    x, w, t = ce_inputs(n, 777, 72, dtype, 0.5, key=1)
    t[0] = 5
    t[n // 2] = IGN
    clean = ce_check(x, w, t, "mean")
    bad = x.clone()
    out = (t == IGN).nonzero()[:, 0]
    for i, v in zip(out.tolist(), [float("nan"), float("inf"), -float("inf"), torch.finfo(x.dtype).min] * n):
        bad[i] = v
    for a, b in zip(clean, ce_check(bad, w, t, "mean")):
        assert torch.equal(a, b)
    t = torch.full_like(t, IGN)
    for red in ("mean", "sum", "none"):
        loss, dx, dw = ce_check(bad, w, t, red)
        assert not bool(loss.any()) and not bool(dx.any()) and not bool(dw.any())
    # another ignored index, inside the vocabulary
    t = torch.randint(0, 4, (n,), generator=gen(8, n), device=DEV)
    a = ops.linear_cross_entropy(x, w, t, ignore_index=2, reduction="none")
    b = ops.linear_cross_entropy(x, w, torch.where(t == 2, IGN, t), reduction="none")
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_ce_extremes(dtype):
    """Confident and hopeless targets, large logits, NaN rows, bad targets."""
    announce("ce extremes", dtype)
    x, w, t = ce_inputs(70, 300, 64, dtype, key=2, std=30.0)
    loss, dx, dw = ce_check(x, w, t, "none")
    assert float(loss.detach().max()) > 50
    x2 = torch.zeros((3, 64), device=DEV, dtype=DT[dtype])
    w2 = torch.zeros((5, 64), device=DEV, dtype=DT[dtype])
    x2[0, 0], x2[1, 0], x2[2, 0] = 20.0, -60.0, 200.0
    w2[1, 0] = 1.0
    t2 = torch.tensor([1, 1, 1], device=DEV)
    loss, dx, dw = ce_check(x2, w2, t2, "none")
    assert abs(float(loss[0]) / (4 * math.exp(-20.0)) - 1) < 0.05     # far below the logits' own step
    assert float(loss[2]) == 0.0
    # a NaN in one row stays in its row of dx; it is in every row of dw
    x, w, t = ce_inputs(40, 300, 64, dtype, key=3)
    good = ops.linear_cross_entropy(x, w, t, reduction="none")
    xn = x.clone()
    xn[7, 3] = float("nan")
    xn.requires_grad_()
    loss = ops.linear_cross_entropy(xn, w, t, reduction="none")
    assert bool(loss[7].isnan()) and int(loss.isnan().sum()) == 1
    keep = torch.arange(40, device=DEV) != 7
    assert torch.equal(loss[keep], good[keep])
    (dxn,) = torch.autograd.grad(loss.sum(), xn)
    assert bool(dxn[7].isnan().all()) and not bool(dxn[keep].isnan().any())
    for bad in (-1, 300, 2 ** 40):
        tb = t.clone()
        tb[3] = bad
        loss = ops.linear_cross_entropy(x, w, tb, reduction="none")
        assert bool(loss[3].isnan()) and int(loss.isnan().sum()) == 1
        assert bool(ops.linear_cross_entropy(x, w, tb).isnan())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_ce_views(dtype):
    """Strided, unaligned and transposed operands against their contiguous copies."""
    announce("ce views", dtype)
    g = gen(9)
    big = torch.randn((400, 700), generator=g, device=DEV).to(DT[dtype])
    t = torch.randint(0, 90, (50,), generator=g, device=DEV)
    cases = [(big[:50, :128], big[100:190, 128:256]), (big[:100:2, 1:130], big[100:280:2, 3:132]),
             (big[:50, 5:69], big[200:290, 8:72]), (big[:128, :50].t(), big[128:256, 100:190].t())]
    for x, w in cases:
        a = ce_check(x, w, t, "mean")
        b = ce_check(x.contiguous(), w.contiguous(), t, "mean")
        for p, q in zip(a, b):
            assert torch.equal(p, q)


def test_ce_one_gradient_and_equal_bits():
    announce("ce needs_input_grad")
    x, w, t = ce_inputs(300, 1000, 128, "bf16", 0.2, key=4)
    loss, dx, dw = ce_check(x, w, t, "mean")
    xg, wg = x.detach().requires_grad_(), w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.linear_cross_entropy(xg, w.detach(), t), xg)[0], dx)
    assert torch.equal(torch.autograd.grad(ops.linear_cross_entropy(x.detach(), wg, t), wg)[0], dw)
    for _ in range(3):
        for a, b in zip((loss, dx, dw), ce_check(x, w, t, "mean")):
            assert torch.equal(a, b)
    e = ops.linear_cross_entropy(x[:0], w, t[:0])
    assert float(e) == 0.0
    xe = x[:0].detach().requires_grad_()
    wg = w.detach().requires_grad_()
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(xe, wg, t[:0]), (xe, wg))
    assert dx.shape == (0, 128) and not bool(dw.any())
    # the per-position losses belong to the caller
    xg = x.detach().requires_grad_()
    per = ops.linear_cross_entropy(xg, w, t, reduction="none")
    a = torch.autograd.grad(per.sum(), xg, retain_graph=True)[0]
    per.detach().zero_()
    assert torch.equal(a, torch.autograd.grad(per, xg, torch.ones_like(per))[0])


@pytest.mark.parametrize("n,vocab,dim", [(20, 90, 33), (130, 400, 64)])
def test_ce_against_differences(n, vocab, dim):
    """The gradient along a direction against the central difference of the loss.
    With step h the difference is off by h^2 / 6 of the third derivative (at
    most max |dz|^3 per unit of loss, dz the logits' change along the direction) and
    by the two losses' errors over 2 h."""
    announce("ce differences", n, vocab, dim)
    x, w, t = ce_inputs(n, vocab, dim, "f32", 0.2, key=5)
    g = gen(10, n)
    xg, wg = x.requires_grad_(), w.requires_grad_()
    grads = torch.autograd.grad(ops.linear_cross_entropy(xg, wg, t, reduction="sum"), (xg, wg))
    x, w = x.detach(), w.detach()
    h = 2.0 ** -7
    for which in (0, 1):
        d = torch.randn((x, w)[which].shape, generator=g, device=DEV)
        ends, tols = [], 0.0
        for sgn in (1, -1):
            a = (x + sgn * h * d, w) if which == 0 else (x, w + sgn * h * d)
            ends.append(ops.linear_cross_entropy(*a, t, reduction="none").double().sum())
            tols += float(Ref(*a, t, torch.ones(n, device=DEV, dtype=torch.float64)).loss_tol.sum())
        dz = (d @ w.t() if which == 0 else x @ d.t()).abs().max(1).values.double()
        tol = tols / (2 * h) + float((h * h / 6 * (2 * dz) ** 3).sum()) + 1e-6
        got, want = float((grads[which].double() * d.double()).sum()), float((ends[0] - ends[1]) / (2 * h))
        print(f"  {got:.6f} {want:.6f} tolerance {tol:.2e}", flush=True)
        assert abs(got - want) <= tol


# ---------------------------------------------------------------------------
# clip_grad_norm
# ---------------------------------------------------------------------------
def clip_ref(ts, max_norm, eps=1e-6):
    norm = math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))
    return norm, min(1.0, max_norm / (norm + eps))


def clip_check(ts, max_norm, **kw):
    norm, c = clip_ref(ts, max_norm)
    keep = [t.clone() for t in ts]
    outs, got = ops.clip_grad_norm(ts, max_norm, **kw)
    assert got.shape == () and got.dtype == torch.float32
    assert abs(float(got) - norm) <= 4 * F * norm
    for t, o in zip(keep, outs):
        assert o.dtype == t.dtype and o.shape == t.shape
        ref = t.double() * c
        within(o, ref, (u(t.dtype) + 12 * F) * ref.abs() + 1e-45 if c < 1 else torch.zeros_like(ref), "values")
    return outs, got


SHAPES = [(3,), (1,), (257, 33), (16384,), (16385,), (70001,), (0,), (128, 128), (5, 5, 5), (999,), (300000,)]


@pytest.mark.parametrize("dtypes", [("f32",), ("bf16",), ("bf16", "f32")])
def test_clip_grad_norm(dtypes):
    announce("clip", dtypes)
    g = gen(11, len(dtypes))
    for max_norm in (1.0, 1e9, 0.0):
        ts = [torch.randn(s, generator=g, device=DEV).to(DT[dtypes[i % len(dtypes)]])
              for i, s in enumerate(SHAPES)]
        keep = [t.clone() for t in ts]
        outs, norm = clip_check(ts, max_norm)
        assert all(torch.equal(a, b) for a, b in zip(ts, keep)), "the gradients changed"
        n2 = ops.global_norm(ts)
        assert torch.equal(n2, norm)
        version = ts[0]._version
        back, n3 = ops.clip_grad_norm(ts, max_norm, out=ts)
        assert torch.equal(n3, norm) and ts[0]._version > version
        assert all(torch.equal(a, b) and a is c for a, b, c in zip(back, outs, ts))


def test_clip_many_and_views():
    """More tensors than one launch takes, on every phase of 16 bytes, results on another phase,
    permuted layouts."""
    announce("clip many")
    g = gen(12)
    for dt in (torch.float32, torch.bfloat16):
        flat = torch.randn(400000, generator=g, device=DEV).to(dt)
        dst = torch.full((400007,), 9.0, device=DEV, dtype=dt)
        ts, os, at = [], [], 0
        for i in range(250):
            k = (i * 37) % 2911 + 1
            ts.append(flat[at:at + k])
            os.append(dst[at + 3:at + 3 + k])
            at += k
        _, norm = clip_check(ts, 2.0, out=os)
        assert bool((dst[:3] == 9).all()) and bool((dst[at + 3:] == 9).all())
        clip_check(ts[:1] * 1, 1e-3)
        clip_check([flat[1:350000]], 0.5)
        p = flat[:24 * 36].view(24, 36).t()
        outs, _ = clip_check([p], 1.0)
        assert outs[0].stride() == p.stride()
        clip_check([flat[:300].view(30, 10)[:, ::2], flat[:4].expand(7, 4)], 0.1)
        a, n1 = ops.clip_grad_norm(ts, 2.0)
        for _ in range(3):
            b, n2 = ops.clip_grad_norm(ts, 2.0)
            assert torch.equal(n1, n2) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_clip_extremes():
    announce("clip extremes")
    for dt in (torch.float32, torch.bfloat16):
        z = torch.zeros(1000, device=DEV, dtype=dt)
        outs, norm = ops.clip_grad_norm([z], 1.0)
        assert float(norm) == 0 and not bool(outs[0].any())
        big = torch.full((1000,), 2.0 ** 100, device=DEV, dtype=dt)       # squares past float32
        outs, norm = ops.clip_grad_norm([big, z], 1.0)
        assert abs(float(norm) / (2.0 ** 100 * math.sqrt(1000)) - 1) < 1e-6
        within(outs[0], torch.full((1000,), 1000 ** -0.5, device=DEV, dtype=torch.float64),
               torch.full((1000,), (u(dt) + 12 * F) / 30, device=DEV, dtype=torch.float64), "big")
        tiny = torch.full((1000,), 2.0 ** -120, device=DEV, dtype=dt)     # squares below float32
        assert abs(float(ops.global_norm([tiny])) / (2.0 ** -120 * math.sqrt(1000)) - 1) < 1e-6
        nan = torch.ones(100, device=DEV, dtype=dt)
        nan[50] = float("nan")
        outs, norm = ops.clip_grad_norm([z, nan], 1.0)
        assert bool(norm.isnan()) and bool(outs[0].isnan().all()) and bool(outs[1].isnan().all())
        nan[50] = float("inf")
        outs, norm = ops.clip_grad_norm([nan], 1.0)
        assert bool(norm.isinf()) and bool(outs[0][50].isnan()) and float(outs[0][0]) == 0.0


# ---------------------------------------------------------------------------
# streams, graphs, large offsets
# ---------------------------------------------------------------------------
def _step(x, w, emb, ids, t):
    h = ops.embedding(ids, emb, scale=1.5)
    loss = ops.linear_cross_entropy(x + h, w, t)
    dx, dw, de = torch.autograd.grad(loss, (x, w, emb))
    (cx, cw, ce), norm = ops.clip_grad_norm([dx, dw, de], 0.01)
    return [loss.detach(), cx, cw, ce, norm]


def _step_inputs(key):
    x, w, t = ce_inputs(300, 1200, 128, "bf16", 0.2, key=key)
    g = gen(13, key)
    emb = torch.randn((500, 128), generator=g, device=DEV).to(torch.bfloat16)
    ids = make_ids(300, 500, "zipf", g)
    return x, w, emb, ids, t


def test_side_stream():
    announce("side stream")
    a = _step_inputs(20)
    for v in a[:3]:
        v.requires_grad_()
    want = _step(*a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _step(*a)
    torch.cuda.current_stream().wait_stream(s)
    for p, q in zip(got, want):
        assert torch.equal(p, q)


def test_graph_capture():
    """A whole step captured and replayed on changing inputs, with eager steps between the
    replays, every replay against the eager result."""
    announce("graph capture")
    static = [v.clone() for v in _step_inputs(21)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        leaves = [v.detach().requires_grad_() for v in static[:3]]
        _step(*leaves, *static[3:])
    torch.cuda.current_stream().wait_stream(s)
    del leaves
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        # leaves of the captured graph only, over the static buffers
        leaves = [v.detach().requires_grad_() for v in static[:3]]
        out = _step(*leaves, *static[3:])
    del leaves
    for r in range(4):
        new = _step_inputs(22 + r)
        for d, v in zip(static, new):
            d.copy_(v)
        for v in new[:3]:
            v.requires_grad_()
        want = _step(*new)
        torch.cuda.synchronize()
        for o in out:
            o.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, want):
            assert torch.equal(p, q), f"replay {r}"


def test_offsets_past_32_bits():
    """A table of more than 2^31 elements (5 GB): rows at its end looked up, scored against and
    given gradients."""
    announce("large offsets")
    vocab, dim, n = 600011, 4096, 6
    w = torch.zeros((vocab, dim), device=DEV, dtype=torch.bfloat16)
    g = gen(14)
    rows = torch.tensor([0, 1, 524287, 524289, vocab - 2, vocab - 1], device=DEV)
    w[rows] = (torch.randn((n, dim), generator=g, device=DEV) / 64).to(torch.bfloat16)
    assert torch.equal(ops.embedding(rows, w), w[rows])
    grad = torch.randn((n, dim), generator=g, device=DEV).to(torch.bfloat16)
    dw = ops.embedding_grad(rows, grad, vocab)
    assert torch.equal(dw[rows], grad)
    dw[rows] = 0
    assert not bool(dw.any())
    del dw
    x = (torch.randn((n, dim), generator=g, device=DEV) + 30 * w[rows].float()).to(torch.bfloat16).requires_grad_()
    w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, rows, reduction="none")
    # all other rows are zero: their logits are 0
    xd, wd = x.detach().double(), w.detach()[rows].double()
    z = xd @ wd.t()
    lse = torch.log(torch.exp(z).sum(1) + (vocab - n))
    ref = lse - z.diagonal()
    tol = 4 * (dim / 4 + 16) * F * (xd.abs() @ wd.abs().t()).max() + F * (200 + vocab / 2000)
    within(loss, ref, tol.expand(n), "loss")
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    p = torch.exp(z - lse[:, None])
    G = p - torch.eye(n, device=DEV, dtype=torch.float64)
    e = u(torch.bfloat16) + float(tol) * 4
    ref = G @ wd
    within(dx, ref, u(torch.bfloat16) * ref.abs() + e * (G.abs() + p) @ wd.abs() + 1e-30, "dx")
    ref = G.t() @ xd
    within(dw[rows], ref, u(torch.bfloat16) * ref.abs() + e * (G.abs() + p).t() @ xd.abs(), "dw")
    other = torch.tensor([2, 300000, 524288, vocab - 3], device=DEV)
    q = torch.exp(-lse)
    ref = (q @ xd).expand(4, dim)
    within(dw[other], ref, u(torch.bfloat16) * ref.abs() + e * (q @ xd.abs()).expand(4, dim), "dw of the rest")
