"""The vocabulary's operators on either side of the sizes at which another kernel, tile or plan
takes over, and their C entry points without what the Python layer always gives.  Formulas and
tolerances are those of test_gpu_vocab."""

import ctypes

import pytest
import torch

from gpu_util import announce
from mamba2_jax import _lib as L
from mamba2_jax import ops
from test_gpu_vocab import DEV, DT, F, IGN, ce_check, ce_inputs, clip_check, gen, grad_ref, make_ids, u, within

pytestmark = pytest.mark.gpu

# tiles of 256 and 128 tokens and their remainders, tokens that the packing finds itself (up to
# 1024) or not, widths of whole K steps or not, several tiles a workgroup, K parts
TILES = [(200, 33000, 64), (300, 33003, 264), (513, 20000, 128), (640, 9000, 520), (1023, 5000, 192), (1024, 5000, 65),
         (1025, 5001, 64), (1100, 40000, 96), (2000, 33000, 128), (4099, 3000, 256), (70, 66000, 700), (257, 700, 2500)]


@pytest.mark.parametrize("n,vocab,dim", TILES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_ce_tiles(n, vocab, dim, dtype):
    announce("ce tiles", n, vocab, dim, dtype)
    masked = [0.0, 0.5, 0.97][(n + vocab + dim) % 3]
    x, w, t = ce_inputs(n, vocab, dim, dtype, masked, key=30)
    ce_check(x, w, t, ["mean", "none"][(n + dim) % 2])


@pytest.mark.parametrize("n,vocab,dtype", [(5000, 60011, "bf16"), (1700, 60011, "f32")])
def test_ce_pieces(n, vocab, dtype):
    """G does not fit its 512 MB: two pieces of the vocabulary, dx added up over them."""
    announce("ce pieces", n, vocab, dtype)
    x, w, t = ce_inputs(n, vocab, 72, dtype, 0.1, key=31)
    t[:40] = torch.arange(vocab - 40, vocab, device=DEV)
    t[40:44] = torch.tensor([0, 30207, 30208, 30209], device=DEV)
    ce_check(x, w, t, "mean")


@pytest.mark.parametrize("n", [70, 1500])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_ce_kept_everywhere(n, dtype):
    """One token kept, wherever it is; none; all but one."""
    announce("ce kept", n, dtype)
    x, w, t = ce_inputs(n, 900, 64, dtype, key=32)
    for at in (0, 63, 64, n - 1):
        one = torch.full_like(t, IGN)
        one[at] = t[at]
        ce_check(x, w, one, "mean")
        rest = t.clone()
        rest[at] = IGN
        ce_check(x, w, rest, "sum")
    ce_check(x, w, torch.full_like(t, IGN), "none")


def _fwd(x, w, t, mean=1, saved=False, **over):
    n, dim = x.shape
    loss, lse = (torch.empty(n, device=DEV) for _ in range(2))
    total = torch.empty((), device=DEV)
    a = L.LinearCrossEntropyArgs(
        x=x.data_ptr(), weight=w.data_ptr(), targets=t.data_ptr(), loss=loss.data_ptr(), lse=lse.data_ptr(),
        total=total.data_ptr(), n=n, vocab=w.shape[0], dim=dim, ldx=x.stride(0), ldw=w.stride(0), ignore_index=IGN,
        dtype=L.dtype_code(w, "w"), target_dtype=L.M2_I64, mean=mean)
    buf = None
    if saved:
        size = L.size_of("m2_linear_cross_entropy_saved_size", a)
        buf = torch.empty(size, dtype=torch.uint8, device=DEV)
        a.saved, a.saved_bytes = buf.data_ptr(), size
    L.call_with_workspace("m2_linear_cross_entropy", a, w.device)
    return loss, lse, total, buf


def _bwd(x, w, t, loss, lse, buf, mean=1, want=(True, True)):
    g = torch.full((1,), 1.5, device=DEV)
    dx, dw = torch.full_like(x, 7.0), torch.full_like(w, 7.0)
    a = L.LinearCrossEntropyGradArgs(
        weight=w.data_ptr(), grad_loss=g.data_ptr(), grad_x=dx.data_ptr() if want[0] else None,
        grad_weight=dw.data_ptr() if want[1] else None, n=x.shape[0], vocab=w.shape[0], dim=x.shape[1],
        ldx=x.stride(0), ldw=w.stride(0), ignore_index=IGN, dtype=L.dtype_code(w, "w"), target_dtype=L.M2_I64, mean=mean)
    if buf is None:
        a.x, a.targets, a.loss, a.lse = x.data_ptr(), t.data_ptr(), loss.data_ptr(), lse.data_ptr()
    else:
        a.saved, a.saved_bytes = buf.data_ptr(), buf.numel()
    L.call_with_workspace("m2_linear_cross_entropy_grad", a, w.device)
    return dx, dw


@pytest.mark.parametrize("n,vocab,dim", [(9, 300, 64), (40, 700, 72), (300, 5000, 136), (1300, 900, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_c_entries_with_and_without_saved(n, vocab, dim, dtype):
    """The gradient from the buffer that the forward leaves, and from its loss and lse alone; loss,
    lse and total of one call."""
    announce("saved", n, vocab, dim, dtype)
    x, w, t = ce_inputs(n, vocab, dim, dtype, 0.3, key=33)
    a, b = _fwd(x, w, t), _fwd(x, w, t, saved=True)
    kept = t != IGN
    z = x.double() @ w.double().t()
    lse = torch.where(kept, torch.logsumexp(z, 1), torch.zeros(n, device=DEV, dtype=torch.float64))
    tol = 4 * (6 if dtype == "f32" else 1) * (dim / 4 + 16) * F * (x.abs().double() @ w.abs().double().t()).max() \
        + F * (200 + 8 * z.abs().max())
    for loss, l, total, _ in (a, b):
        within(l, lse, tol.expand(n), "lse")
        assert not bool(loss[~kept].any()) and not bool(l[~kept].any())
        assert abs(float(total) - float(loss.double().sum() / kept.sum())) <= 2 * F * float(total)
    # few tokens are scored by another kernel than they are trained by
    within(a[0], b[0].double(), (2 * tol).expand(n), "losses of both")
    p, q = _bwd(x, w, t, b[0], b[1], None), _bwd(x, w, t, None, None, b[3])
    for v, r in zip(p, q):
        assert torch.equal(v, r)
    dx, _ = _bwd(x, w, t, None, None, b[3], want=(True, False))
    _, dw = _bwd(x, w, t, None, None, b[3], want=(False, True))
    assert torch.equal(dx, p[0]) and torch.equal(dw, p[1])


GRADS = [(255, 5000, 72, "zipf"), (256, 5000, 72, "same"), (256, 9, 1, "any"), (257, 5000, 72, "zipf"),
         (256, 300, 2056, "zipf"), (200, 7, 3, "any"), (1024, 300, 64, "zipf"), (1025, 300, 7, "zipf"),
         (4097, 262142, 8, "zipf"), (4097, 262143, 8, "zipf"), (300, 262144, 9, "any"), (16385, 2000, 33, "zipf"),
         (16384, 300, 520, "same"), (700, 40, 4097, "zipf")]


@pytest.mark.parametrize("n,vocab,dim,how", GRADS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_embedding_grad_sizes(n, vocab, dim, how, dtype):
    announce("embedding_grad sizes", n, vocab, dim, how, dtype)
    g = gen(34, n, vocab, dim)
    ids = make_ids(n, vocab, how, g)
    ids[n // 2] = vocab                              # takes no part
    grad = torch.randn((n, dim), generator=g, device=DEV).to(DT[dtype])
    for padding in (None, int(ids[0])):
        ref, mag, cnt = grad_ref(ids, grad, vocab, 2.5, padding)
        tol = u(grad.dtype) * ref.abs() + (cnt + 3) * F * mag * 1.01 + 1e-45 * (cnt > 0)
        out = ops.embedding_grad(ids, grad, vocab, scale=2.5, padding_idx=padding)
        within(out, ref, tol, "rows")
        assert torch.equal(out, ops.embedding_grad(ids, grad, vocab, scale=2.5, padding_idx=padding))
        # into rows of a wider tensor, unaligned, the others untouched
        wide = torch.randn((vocab, dim + 3), generator=g, device=DEV).to(DT[dtype])
        view, before = wide[:, 1:1 + dim], wide.clone()
        ops.embedding_grad(ids, grad, vocab, scale=2.5, padding_idx=padding, out=view)
        want = before[:, 1:1 + dim].double() + ref
        within(view, want, u(grad.dtype) * want.abs() + F * before[:, 1:1 + dim].double().abs()
               + (cnt + 4) * F * mag * 1.01, "added")
        assert torch.equal(wide[:, 0], before[:, 0]) and torch.equal(wide[:, 1 + dim:], before[:, 1 + dim:])
        unnamed = cnt[:, 0] == 0
        assert torch.equal(wide[unnamed], before[unnamed])


@pytest.mark.parametrize("dim", [1, 2, 3, 5, 7, 8, 9, 15, 17, 511, 513, 1025])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_embedding_widths(dim, dtype):
    announce("embedding widths", dim, dtype)
    g = gen(35, dim)
    w = torch.randn((50, dim + 1), generator=g, device=DEV).to(DT[dtype])
    ids = torch.randint(0, 50, (300,), generator=g, device=DEV)
    for v in (w[:, :dim], w[:, 1:]):
        assert torch.equal(ops.embedding(ids, v), v[ids])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_clip_large(dtype):
    """More than the last-level cache takes, on odd offsets, in place and not."""
    announce("clip large", dtype)
    g = gen(36)
    flat = torch.randn(80_000_003, generator=g, device=DEV).to(DT[dtype])
    ts = [flat[1:3], flat[3:70_000_001], flat[70_000_001:70_000_002], flat[70_000_002:]]
    outs, norm = clip_check(ts, 3.0)
    back, n2 = ops.clip_grad_norm(ts, 3.0, out=ts)
    assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(outs, back))
    # by single elements: the result on another phase than its tensor
    dst = torch.empty(1_000_001, device=DEV, dtype=DT[dtype])
    clip_check([flat[:1_000_000]], 0.5, out=[dst[1:]])


def test_second_derivative_is_refused():
    announce("second derivative")
    x, w, t = ce_inputs(20, 90, 64, "f32", key=37)
    x.requires_grad_()
    (dx,) = torch.autograd.grad(ops.linear_cross_entropy(x, w, t), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)


def test_weight_changed_before_the_gradient_is_refused():
    announce("version")
    x, w, t = ce_inputs(20, 90, 64, "bf16", key=38)
    w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, t)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, w)
    # x is not read again: changing it changes nothing
    xg = x.clone().requires_grad_()
    w2 = w.detach()
    want = torch.autograd.grad(ops.linear_cross_entropy(xg, w2, t), xg)[0]
    loss = ops.linear_cross_entropy(xg, w2, t)
    with torch.no_grad():
        xg.zero_()
    assert torch.equal(torch.autograd.grad(loss, xg)[0], want)


@pytest.mark.parametrize("n", [3, 60, 300, 700])
def test_ce_target_is_not_rounded(n):
    """bfloat16: G at the target, most of a row's weight, rounds by up to 2^-8 of it in every column
    alike, which dx (and dw of up to 64 tokens) gets back.  What is left are roundings of
    either sign, each at most 2^-8 of its term: their sum over a row's columns with the
    results' signs exceeds 6 times the root of the sum of their squares' bounds once in
    3e7 rows (Hoeffding), where the one lost would be 2^-8 of the sum of all.  (The results' own
    roundings have either sign where a row is a sum of several: dw of three tokens is nearly
    one row of x times a number, whose roundings all depend on that number.)"""
    announce("ce target", n)
    dim, vocab, up = 2048, 1500, 1.0038          # 1.0038: a rounding of nearly half a step
    g = gen(39, n)
    w = (torch.randn((vocab, dim), generator=g, device=DEV) / dim ** 0.5).to(torch.bfloat16)
    x = torch.randn((n, dim), generator=g, device=DEV).to(torch.bfloat16)
    t = torch.randperm(vocab, generator=g, device=DEV)[:n]
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = ops.linear_cross_entropy(xg, wg, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (xg, wg), torch.tensor(up, device=DEV))
    X, W = x.double(), w.double()
    z = X @ W.t()
    G = torch.softmax(z, 1)
    G[torch.arange(n, device=DEV), t] -= 1
    G *= float(torch.tensor(up))
    rounded = G.clone()
    rounded[torch.arange(n, device=DEV), t] = 0              # the target's is not
    e = 1e-4                                                 # the logits' and lse's errors, relative to a term
    ub = 2.0 ** -8

    def check(got, a, b, c, what):
        ref = a @ b
        s = ((got.double() - ref) * ref.sign()).sum(1).abs()
        bound = 6 * ub * ((ref ** 2).sum(1).sqrt() + ((c ** 2) @ (b ** 2)).sum(1).sqrt()) \
            + (e + ub ** 2) * (a.abs() @ b.abs()).sum(1)
        print(f"  {what}: worst {float((s / bound).max()):.3f} of the bound", flush=True)
        assert bool((s <= bound).all())
        lost = ub * 0.9 * ref.abs().sum(1)
        assert bool((lost > 2 * bound).all()), "the bound would not notice"
    check(dx, G, W, rounded, "dx")
    if n == 60:
        check(dw[t], G.t()[t], X, rounded.t()[t], "dw")


@pytest.mark.parametrize("vocab", [1, 126, 255, 511, 512, 16383, 20000, 65535, 65536, 262142])
@pytest.mark.parametrize("n", [1023, 2047, 2048, 2049, 4097, 8191, 8192, 8193, 12288, 12289, 16383])
def test_embedding_grad_sorts(n, vocab):
    """Whole numbers, whose sums are exact: every entry is added once, to its row."""
    announce("embedding_grad sorts", n, vocab)
    g = gen(35, n, vocab)
    ids = make_ids(n, vocab, "any" if n & 1 else "zipf", g)
    ids[n // 3] = vocab
    ids[n // 2] = -1
    grad = torch.randint(-100, 101, (n, 4), generator=g, device=DEV).float()
    want = torch.zeros(vocab + 1, 4, dtype=torch.float64, device=DEV)
    want.index_add_(0, torch.where((ids < 0) | (ids > vocab), vocab, ids).long(), grad.double())
    assert torch.equal(ops.embedding_grad(ids, grad, vocab).double(), want[:vocab])


@pytest.mark.parametrize("n", [60, 700])
def test_ce_target_each_loss(n):
    """The same for a gradient of each loss, which G holds: dx gets back what rounding takes from
    G at the target (the bound of test_ce_target's docstring: roundings of either sign)."""
    announce("ce target, each loss", n)
    dim, vocab = 2048, 1500
    g = gen(40, n)
    w = (torch.randn((vocab, dim), generator=g, device=DEV) / dim ** 0.5).to(torch.bfloat16)
    x = torch.randn((n, dim), generator=g, device=DEV).to(torch.bfloat16)
    t = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    up = torch.full((n,), 1.0038, device=DEV)
    xg = x.clone().requires_grad_()
    dx, = torch.autograd.grad(ops.linear_cross_entropy(xg, w, t, reduction="none"), xg, up)
    G = torch.softmax(x.double() @ w.double().t(), 1)
    G[torch.arange(n, device=DEV), t] -= 1
    G *= up.double()[:, None]
    rounded = G.clone()
    rounded[torch.arange(n, device=DEV), t] = 0
    W, ub = w.double(), 2.0 ** -8
    ref = G @ W
    s = ((dx.double() - ref) * ref.sign()).sum(1).abs()
    bound = 6 * ub * ((ref ** 2).sum(1).sqrt() + ((rounded ** 2) @ (W ** 2)).sum(1).sqrt()) \
        + (1e-4 + ub ** 2) * (G.abs() @ W.abs()).sum(1)
    assert bool((s <= bound).all())
    assert bool((0.9 * ub * ref.abs().sum(1) > 2 * bound).all()), "the bound would not notice"


@pytest.mark.parametrize("n", [484, 600, 1210])
@pytest.mark.parametrize("how", ["mean", "sum"])
def test_ce_dw_one_gradient(n, how):
    """bfloat16, one gradient for all losses: it is not part of what G rounds.  With zero
    weights every logit is 0 and softmax 1 / 4096; rows of x cancel in pairs, so a target's row
    of dw is its row of x times -up, up to 2^-12 by the rounding of -1 + 1 / 4096.  One
    rounding of the result is left (2^-8), and float32's of sums over the tokens."""
    announce("ce dw one gradient", n, how)
    vocab, dim = 4096, 264
    up = 1.0351 * (n if how == "mean" else 1)          # of each loss 1.0351: a rounding of nearly half a step
    g = gen(41, n)
    half = torch.randn((n // 2, dim), generator=g, device=DEV).to(torch.bfloat16)
    x = torch.cat([half, -half])
    w = torch.zeros((vocab, dim), device=DEV, dtype=torch.bfloat16, requires_grad=True)
    t = torch.randperm(vocab, generator=g, device=DEV)[:n]
    dw, = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, reduction=how), w, torch.tensor(up, device=DEV))
    each = float(torch.tensor(up)) / (n if how == "mean" else 1)
    ref = torch.zeros((vocab, dim), dtype=torch.float64, device=DEV)
    ref[t] = -each * x.double()
    small = (n + 8) * 2.0 ** -24 * each * (x.double().abs().sum(0) / vocab)
    tol = ref.abs() * (2.0 ** -8 + 2.0 ** -12 + 2.0 ** -16) + small
    assert bool(((dw.double() - ref).abs() <= tol).all())
    once = torch.tensor(each * (1 - 1 / vocab), device=DEV).bfloat16().double()      # rounded before x
    assert bool((((-once * x.double()).bfloat16().double() - ref[t]).abs() > tol[t]).any()), "would not be noticed"
