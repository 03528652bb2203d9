"""The gated linear recurrence, its gradient and its single step against the formulas in 64 bits.

Tolerances are per element and derived from the arithmetic; F = 2^-24, u(T) half a step of T.

* A gate q = sigmoid(r) is off by (6 + 2 |r|) F of itself: the argument's product rounds by |r| F, the
  exponential and the reciprocal by two steps each, the sum by half a one.
* L = A q by F more; alpha = 1 - exp(L) by 12 F more (the polynomial's seven roundings; below -0.35 the
  exponential's 2 F over alpha > 0.29, with the argument's |L| F a where a is its weight); beta by half of
  alpha's and 5 F, and so is 1 / beta; what is added, b = beta s x, by the sum of its factors' and 2 F.
* A step passes its state's error on by a and adds alpha's error times the state, b's and two roundings of
  what it adds up; the joins of maps (a product and a sum for each of at most 16 lane and wavefront
  levels, and P, whose exponent sums 4 terms) add up to 24 F of the sum of the magnitudes.
  So the error obeys the recurrence itself, run here on magnitudes; and from the end for l.
* A gradient is a product: its factors' errors, times the other factors' magnitudes.
* What is stored in bfloat16 is off by u of itself, gradients from a sum over n by n F of the magnitudes.
"""

import zlib

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
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(key).encode()))


def within(got, want, tol, what):
    got = got.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol) & ~(got.isnan() & want.isnan())
    worst = float(((got - want).abs() / tol.clamp_min(1e-300)).nan_to_num(0.0).max()) if got.numel() else 0.0
    print(f"  {what}: worst error / tolerance {worst:.3f}", flush=True)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the tolerance"


def scan(a, b):
    """y[t] = a[t] y[t - 1] + b[t] along dimension 1, y[-1] = 0; a of 0 forgets whatever came before"""
    y = torch.empty_like(b)
    at = torch.zeros_like(b[:, 0])
    for t in range(b.shape[1]):
        at = torch.where(a[:, t] == 0, b[:, t], a[:, t] * at + b[:, t])
        y[:, t] = at
    return y


class Reference:
    """Results in 64 bits and what a kernel may be off by, of h, last and (with g) the gradients."""

    def __init__(self, x, r, i, A, h0, seq, g=None, glast=None):
        x, r, i, A = (t.detach().double() for t in (x, r, i, A))
        b, n, d = x.shape
        live = torch.ones((b, n, 1), dtype=torch.bool, device=x.device)
        clear = torch.zeros_like(live)
        if seq is not None:
            live = (seq >= 0)[..., None]
            clear[:, 1:, 0] = (seq[:, 1:] != seq[:, :-1]) & (seq[:, 1:] >= 0)
        zero = torch.zeros_like(x)
        x, r, i = (torch.where(live, t, zero) for t in (x, r, i))
        q, s = torch.sigmoid(r), torch.sigmoid(i)
        eq, es = (6 + 2 * r.abs()) * F, (6 + 2 * i.abs()) * F
        la = A * q
        alpha = -torch.expm1(la)
        ea = eq + 13 * F
        beta = torch.sqrt(-torch.expm1(2 * la))
        eb = ea / 2 + 5 * F
        add = torch.where(live, beta * s * x, zero)
        a = torch.where(clear, zero, torch.where(live, torch.exp(la), zero + 1))
        alpha_live = torch.where(live & ~clear, alpha, zero)
        eadd = (eb + es + 2 * F) * add.abs()
        h0 = zero[:, 0] if h0 is None else h0.detach().double()
        first = lambda t, v: torch.cat([t[:, :1] + a[:, :1] * v[:, None], t[:, 1:]], 1)
        before = lambda t, v: torch.where(clear, zero, torch.cat([v[:, None], t[:, :-1]], 1))
        h = scan(a, first(add, h0))
        mag = scan(a, first(add.abs(), h0.abs()))
        mb = before(mag, h0.abs())
        eh = scan(a, alpha_live * ea * mb + eadd + 2 * F * (mb + add.abs() + mag)) + 24 * F * mag
        self.h, self.last = torch.where(live, h, zero), h[:, -1]
        self.eh, self.elast = torch.where(live, eh, zero), eh[:, -1]
        if g is None:
            return
        g = torch.where(live, g.detach().double(), zero)
        # the last position's gradient is a sum, whose terms a kernel may pass on apart from each other (a g and
        # a glast, each rounded): of magnitude |g| + |glast|, however much of it cancels
        gl = torch.zeros_like(g[:, 0]) if glast is None else glast.detach().double()
        gmag = torch.cat([g[:, :-1].abs(), g[:, -1:].abs() + gl.abs()[:, None]], 1)
        g = torch.cat([g[:, :-1], g[:, -1:] + gl[:, None]], 1)
        later = torch.cat([a[:, 1:], zero[:, :1]], 1)
        lam = scan(later.flip(1), g.flip(1)).flip(1)
        lmag = scan(later.flip(1), gmag.flip(1)).flip(1)
        passed = (alpha_live * ea * lmag + 3 * F * lmag)
        passed = torch.cat([passed[:, 1:], zero[:, :1]], 1)
        el = scan(later.flip(1), (passed + 2 * F * lmag).flip(1)).flip(1) + 24 * F * lmag
        self.dh0 = a[:, 0] * lam[:, 0]
        self.edh0 = a[:, 0] * el[:, 0] + passed[:, 0] + (alpha_live * ea * lmag)[:, 0] + 4 * F * lmag[:, 0]
        lam, lmag, el = (torch.where(live, t, zero) for t in (lam, lmag, el))
        p, ep = before(h, h0), before(eh, zero[:, 0])
        root = torch.where(beta > 0, beta, zero + 1)
        rise = torch.where(beta > 0, torch.exp(2 * la) / root * s * x, zero)
        ea1 = torch.exp(la)
        self.dx = lam * beta * s
        self.edx = el * beta * s + lmag * beta * s * (eb + es + 3 * F)
        self.di = self.dx * x * (1 - s)
        self.edi = (self.edx + lmag * beta * s * (es + 5 * F)) * x.abs() * (1 - s)
        dL = lam * (ea1 * p - rise)
        aerr = alpha * ea + 2 * F                   # of a = 1 - alpha
        edL = el * (ea1 * p - rise).abs() + lmag * (
            ea1 * ep + aerr * mb + rise.abs() * (eb + es + 8 * F) + 2 * aerr * (rise / ea1.clamp_min(1e-30)).abs()
            + 4 * F * (ea1 * mb + rise.abs()))
        edL = torch.where(live, edL, zero)
        slope = (la * (1 - q)).abs()
        self.dr, self.edr = dL * la * (1 - q), (edL + dL.abs() * (2 * eq + 6 * F)) * slope
        terms = torch.where(live, dL * q, zero)
        self.dA = terms.sum((0, 1))
        self.edA = (edL * q + terms.abs() * (eq + 2 * F)).sum((0, 1)) + b * n * F * terms.abs().sum((0, 1))
        self.dr, self.edr = (torch.where(live, t, zero) for t in (self.dr, self.edr))


def inputs(batch, seqlen, dim, dtype, fused=False, packed=0, carried=False, low=1e-3, high=0.5):
    g = gen("rec", batch, seqlen, dim, packed)
    dt = DT[dtype]
    if fused:
        x, r, i = (t.detach() for t in torch.randn((batch, seqlen, 3 * dim), generator=g, device=DEV).to(dt).split(dim, 2))
    else:
        x, r, i = (torch.randn((batch, seqlen, dim), generator=g, device=DEV).to(dt) for _ in range(3))
    A = -torch.exp(torch.empty(dim, device=DEV).uniform_(0, 1, generator=g) *
                   torch.log(torch.tensor(high / low)) + torch.log(torch.tensor(low)))
    h0 = torch.randn((batch, dim), generator=g, device=DEV) if carried else None
    seq = None
    if packed:
        starts = torch.rand((batch, seqlen), generator=g, device=DEV) < 1.0 / packed
        seq = starts.cumsum(1).int()
        pad = torch.rand((batch, seqlen), generator=g, device=DEV) < 0.1
        seq[pad] = -1
        seq[0, seqlen - seqlen // 3:] = -1
    go = torch.randn((batch, seqlen, dim), generator=g, device=DEV).to(dt)
    gl = torch.randn((batch, dim), generator=g, device=DEV)
    return x, r, i, A, h0, seq, go, gl


def check(x, r, i, A, h0, seq, go, gl):
    dt = x.dtype
    leaves = [t.clone().requires_grad_() if t.is_contiguous() else t.detach().requires_grad_() for t in (x, r, i, A)]
    if h0 is not None:
        leaves.append(h0.clone().requires_grad_())
    want = Reference(x, r, i, A, h0, seq, go, gl)
    with torch.no_grad():
        h, last = ops.gated_linear_recurrence(x, r, i, A, h0, seq, True)
        alone = ops.gated_linear_recurrence(x, r, i, A, h0, seq)
    assert h.dtype == dt and last.dtype == torch.float32 and h.is_contiguous() and torch.equal(h, alone)
    within(h, want.h, want.eh + u(dt) * want.h.abs() + 1e-38, "h")
    within(last, want.last, want.elast + 1e-38, "last")
    h2, last2 = ops.gated_linear_recurrence(*leaves[:4], leaves[4] if h0 is not None else None, seq, True)
    assert torch.equal(h2, h) and torch.equal(last2, last)
    grads = torch.autograd.grad((h2, last2), leaves, (go, gl), retain_graph=True)
    for name, got in zip(("dx", "dr", "di", "dA", "dh0"), grads):
        ref, tol = getattr(want, name), getattr(want, "e" + name)
        within(got, ref, tol + (u(got.dtype) * ref.abs() if got.dtype == torch.bfloat16 else 0) + 1e-37, name)
    again = torch.autograd.grad((h2, last2), leaves, (go, gl))
    assert all(torch.equal(p, q) for p, q in zip(grads, again))
    return grads


SIZES = [(1, 1, 1), (2, 1, 5), (1, 2, 3), (3, 3, 2), (2, 5, 4), (1, 63, 17), (2, 64, 64), (1, 65, 65), (2, 127, 1),
         (1, 128, 130), (1, 200, 1001), (3, 257, 36), (1, 515, 16), (2, 300, 260), (1, 1030, 3)]


@pytest.mark.parametrize("batch,seqlen,dim", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("fused,packed,carried", [(False, 0, False), (True, 0, True), (True, 20, True), (False, 3, False)])
def test_recurrence(batch, seqlen, dim, dtype, fused, packed, carried):
    announce("recurrence", batch, seqlen, dim, dtype, fused, packed, carried)
    check(*inputs(batch, seqlen, dim, dtype, fused, packed, carried))


# rows of one segment and of many, of one and of several tiles, ended inside a tile
LARGE = [(8, 300, 640), (1, 2100, 700), (2, 900, 2560), (16, 70, 5120), (6, 333, 4500), (1, 5000, 2560)]


@pytest.mark.parametrize("batch,seqlen,dim", LARGE)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("packed", [0, 100])
def test_recurrence_large(batch, seqlen, dim, dtype, packed):
    announce("recurrence large", batch, seqlen, dim, dtype, packed)
    check(*inputs(batch, seqlen, dim, dtype, True, packed, True))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_recurrence_past_the_cache(dtype):
    """More than the last-level cache holds."""
    announce("past the cache", dtype)
    check(*inputs(7, 1200, 4160, dtype, carried=True))


@pytest.mark.parametrize("low,high", [(1e-6, 1e-5), (1e-4, 1e-3), (0.3, 0.4), (5.0, 60.0)])
def test_recurrence_memories(low, high):
    """From states that keep everything to states that forget at once."""
    announce("memories", low, high)
    check(*inputs(2, 700, 40, "f32", low=low, high=high, carried=True))


def test_recurrence_saturated_gates():
    """Gates at and far past their ends, infinities among them: a of 1 exactly (the root's slope is left
    out) and of exp(A); a constant a near 1, whose rounding would add up over the steps."""
    announce("saturated")
    x, r, i, A, h0, _, go, gl = inputs(1, 400, 24, "f32", carried=True, low=1e-5, high=1e-3)
    for k, v in enumerate((30.0, 300.0, -30.0, -300.0, float("inf"), float("-inf"))):
        r[:, :, 4 * k:4 * k + 2] = v
        i[:, :, 4 * k + 2:4 * k + 4] = v
    want = Reference(x, r.clamp(-1e4, 1e4), i.clamp(-1e4, 1e4), A, h0, None, go, gl)
    # (the gates' bounds above grow with |r|: here they are at most two steps off, as their ends are exact)
    fixed = Reference(x, r.clamp(-8, 8), i.clamp(-8, 8), A, h0, None, go, gl)
    leaves = [t.clone().requires_grad_() for t in (x, r, i, A, h0)]
    h, last = ops.gated_linear_recurrence(*leaves, None, True)
    within(h, want.h, fixed.eh * 2 + 1e-30, "h")
    grads = torch.autograd.grad((h, last), leaves, (go, gl))
    assert all(bool(t.isfinite().all()) for t in grads)
    for name, got in zip(("dx", "di", "dh0"), (grads[0], grads[2], grads[4])):
        mag = getattr(want, name).abs()
        within(got, getattr(want, name), 2000 * F * mag.max() + 0 * mag, name)
    # a closed gate keeps its state for good
    closed = [v for k in (2, 3, 5) for v in (4 * k, 4 * k + 1)]
    assert torch.equal(last[:, closed[2:]], h0[:, closed[2:]])


def test_recurrence_masked_places():
    """What padding holds reaches nothing, and neither does a sequence reach the next one."""
    announce("masked places")
    for dtype in ("f32", "bf16"):
        x, r, i, A, h0, _, go, gl = inputs(3, 260, 37, dtype, carried=True)
        seq = torch.zeros((3, 260), dtype=torch.int64, device=DEV)
        seq[0, 100:] = 1
        seq[0, 200:] = -1
        seq[1] = -5                                    # a row of padding alone
        seq[2, :30] = -1
        seq[2, 131:140] = -2
        clean = check(x, r, i, A, h0, seq, go, gl)
        pad = seq < 0
        dirty = [t.clone() for t in (x, r, i)]
        for t, v in zip(dirty, (float("nan"), float("inf"), float("nan"))):
            t[pad] = v
        g2 = go.clone()
        g2[pad] = float("nan")
        leaves = [t.requires_grad_() for t in (*dirty, A.clone(), h0.clone())]
        h, last = ops.gated_linear_recurrence(*leaves, seq, True)
        assert not bool(h[pad].any())
        assert torch.equal(last[1], h0[1])             # carried past padding to the end
        for p, q in zip(torch.autograd.grad((h, last), leaves, (g2, gl)), clean):
            assert torch.equal(p, q)
        # a NaN in the first sequence of row 0 stays there, forward and backward
        leaves[0].detach()[0, 50, 3] = float("nan")
        h, last = ops.gated_linear_recurrence(*leaves, seq, True)
        assert bool(h[0, 50:100, 3].isnan().all()) and not bool(h[0, 100:].isnan().any())
        g3 = go.clone()
        g3[0, 150, 5] = float("nan")
        dx = torch.autograd.grad((h, last), leaves, (g3, gl))[0]
        assert bool(dx[0, 100:151, 5].isnan().all()) and not bool(dx[0, :100, 5].isnan().any())


def test_recurrence_infinite_state():
    """An infinite state decays to nothing only by a sequence's end."""
    announce("infinite state")
    x, r, i, A, h0, _, go, gl = inputs(2, 90, 8, "f32", carried=True)
    h0[0, 2], h0[1, 3] = float("inf"), float("nan")
    seq = torch.zeros((2, 90), dtype=torch.int32, device=DEV)
    seq[:, 70:] = 1
    h = ops.gated_linear_recurrence(x, r, i, A, h0, seq)
    assert bool((h[0, :70, 2] == float("inf")).all()) and bool(h[1, :70, 3].isnan().all())
    assert bool(h[:, 70:].isfinite().all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_recurrence_layouts(dtype):
    """Strides and alignments: equal inputs of any layout give equal bits."""
    announce("layouts", dtype)
    x, r, i, A, h0, seq, go, gl = inputs(3, 150, 50, dtype, packed=30, carried=True)
    want = ops.gated_linear_recurrence(x, r, i, A, h0, seq, True)
    wide = torch.zeros((3, 150, 173), device=DEV, dtype=x.dtype)
    views = []
    for k, t in enumerate((x, r, i)):
        v = wide[:, :, 3 + 53 * k:53 + 53 * k]
        v.copy_(t)
        views.append(v)
    time_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, r, i)]
    channels_apart = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (x, r, i)]
    steps = [torch.stack([t, t], 2).reshape(3, 300, 50)[:, ::2] for t in (x, r, i)]
    for x2, r2, i2 in (views, time_first, channels_apart, steps):
        got = ops.gated_linear_recurrence(x2, r2, i2, A.double().float(), h0, seq.long(), True)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        leaves = [t.detach().requires_grad_() for t in (x2, r2, i2)]
        plain = [t.detach().requires_grad_() for t in (x, r, i)]
        go2 = go.transpose(0, 1).contiguous().transpose(0, 1)
        p = torch.autograd.grad(ops.gated_linear_recurrence(*leaves, A, h0, seq), leaves, go2)
        q = torch.autograd.grad(ops.gated_linear_recurrence(*plain, A, h0, seq), plain, go)
        assert all(torch.equal(a, b) for a, b in zip(p, q))
    # one row and one step for all, and a gradient that all positions share
    xe, re, ie = x[:1, :1].expand(3, 150, 50), r[:1].expand(3, 150, 50), i[:, :1].expand(3, 150, 50)
    got = ops.gated_linear_recurrence(xe, re, ie, A, h0, seq)
    assert torch.equal(got, ops.gated_linear_recurrence(xe.contiguous(), re.contiguous(), ie.contiguous(), A, h0, seq))
    xl = x.detach().requires_grad_()
    (p,) = torch.autograd.grad(ops.gated_linear_recurrence(xl, r, i, A, h0, seq).sum(), xl)
    (q,) = torch.autograd.grad(ops.gated_linear_recurrence(xl, r, i, A, h0, seq), xl, torch.ones_like(x))
    assert torch.equal(p, q)


def test_recurrence_one_position():
    """A single position has no next one: whatever its stride, forward and backward."""
    announce("one position")
    x, r, i, A, h0, _, go, _ = inputs(3, 1, 50, "bf16", carried=True)
    views = []
    for t in (x, r, i, go):
        for stride in (2 ** 21 + 1, 7):
            v = torch.empty(3 * 50, device=DEV, dtype=x.dtype).as_strided((3, 1, 50), (50, stride, 1))
            v.copy_(t)
            views.append(v)
    want_in = [t.detach().requires_grad_() for t in (x, r, i)]
    want = ops.gated_linear_recurrence(*want_in, A, h0)
    for k in (0, 1):
        leaves = [t.detach().requires_grad_() for t in views[k:6:2]]
        got = ops.gated_linear_recurrence(*leaves, A, h0)
        assert torch.equal(got, want)
        for p, q in zip(torch.autograd.grad(got, leaves, views[6 + k]), torch.autograd.grad(want, want_in, go, retain_graph=True)):
            assert torch.equal(p, q)


@pytest.mark.parametrize("batch,seqlen,dim", [(1, 3001, 65), (1, 2999, 1409), (3, 1025, 4161), (130, 129, 1), (3, 128, 130), (3, 129, 130)])
@pytest.mark.parametrize("packed", [0, 400])
def test_recurrence_segments(batch, seqlen, dim, packed):
    """Segments of every length, of few and of many chains, whose last slab has a single channel; and the same bits
    every time, with other work beside it."""
    announce("segments", batch, seqlen, dim, packed)
    x, r, i, A, h0, seq, go, gl = sets = inputs(batch, seqlen, dim, "f32", packed=packed, carried=True)
    check(*sets)
    want = ops.gated_linear_recurrence(x, r, i, A, h0, seq, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        with torch.cuda.stream(side):
            other = ops.gated_linear_recurrence(x, r, i, A, h0, seq, True)
        got = ops.gated_linear_recurrence(x, r, i, A, h0, seq, True)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want)) and all(torch.equal(p, q) for p, q in zip(other, want))


@pytest.mark.parametrize("packed", [0, 300])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_recurrence_more_rows_than_run_at_once(dtype, packed):
    """Rows that are cut so that no CU idles at the end: what goes back from segment to segment, and the same bits every time."""
    announce("more rows", dtype, packed)
    sets = inputs(9, 1100, 3713, dtype, packed=packed, carried=True)
    check(*sets)
    x, r, i, A, h0, seq, go, gl = sets

    def run():
        leaves = [t.detach().requires_grad_() for t in (x, r, i, A, h0)]
        return torch.autograd.grad(ops.gated_linear_recurrence(*leaves, seq, True), leaves, (go, gl))

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            other = run()
        got = run()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want)) and all(torch.equal(p, q) for p, q in zip(other, want))


def test_recurrence_any_not_a_number():
    """NaNs of all bits (and of all ones, which stand for what is not known yet) go on like any value."""
    announce("any NaN")
    x, r, i, A, h0, _, _, _ = inputs(2, 1500, 70, "f32", carried=True)
    for bits in (-1, 0x7fc00000, 0x7f800001):
        for where in (x, r, i, h0):
            t = where.clone()
            place = (0, 5) if where is h0 else (0, 300, 5)
            t.view(torch.int32)[place] = bits
            assert bool(t[place].isnan())
            h = ops.gated_linear_recurrence(*(t if where is q else q for q in (x, r, i)), A, t if where is h0 else h0)
            after = 0 if where is h0 else 300
            assert bool(h[0, after:, 5].isnan().all())
            h[0, after:, 5] = 0
            assert bool(h.isfinite().all())


def test_recurrence_parameter_types():
    """A and the states in bfloat16: their gradients come back in it."""
    announce("parameter types")
    x, r, i, A, h0, _, go, gl = inputs(2, 70, 12, "bf16", carried=True)
    A16, h16 = A.bfloat16().requires_grad_(), h0.bfloat16().requires_grad_()
    h, last = ops.gated_linear_recurrence(x, r, i, A16, h16, None, True)
    ref = ops.gated_linear_recurrence(x, r, i, A16.detach().float(), h16.detach().float(), None, True)
    assert torch.equal(h, ref[0]) and torch.equal(last, ref[1])
    dA, dh0 = torch.autograd.grad((h, last), (A16, h16), (go, gl))
    assert dA.dtype == dh0.dtype == torch.bfloat16 and dA.shape == (12,) and dh0.shape == (2, 12)


def test_recurrence_only_one_output_used():
    announce("one output")
    x, r, i, A, h0, seq, go, gl = inputs(2, 130, 20, "f32", packed=40, carried=True)
    leaves = [t.clone().requires_grad_() for t in (x, r, i, A, h0)]
    h, last = ops.gated_linear_recurrence(*leaves, seq, True)
    zero = torch.zeros_like(h)
    for got, want in zip(torch.autograd.grad(last, leaves, gl, retain_graph=True),
                         torch.autograd.grad((h, last), leaves, (zero, gl), retain_graph=True)):
        assert torch.equal(got, want)
    for got, want in zip(torch.autograd.grad(h, leaves, go, retain_graph=True),
                         torch.autograd.grad((h, last), leaves, (go, torch.zeros_like(last)))):
        assert torch.equal(got, want)


def test_recurrence_differences():
    """The gradients against differences of the operator itself along random directions: a central
    difference of step e is off by e^2 / 6 of the third derivative (a few hundred here) and by the
    float32 sums' errors over e."""
    announce("differences")
    x, r, i, A, h0, seq, go, gl = inputs(2, 120, 9, "f32", packed=50, carried=True, low=0.05, high=0.5)
    leaves = [t.clone().requires_grad_() for t in (x, r, i, A, h0)]
    run = lambda ts: ops.gated_linear_recurrence(*ts, seq, True)
    loss = lambda o: float((o[0].double() * go.double()).sum() + (o[1].double() * gl.double()).sum())
    grads = torch.autograd.grad(run(leaves), leaves, (go, gl))
    want = Reference(x, r, i, A, h0, seq, go, gl)
    noise = float((want.eh * go.double().abs()).sum() + (want.elast * gl.double().abs()).sum())
    g = gen("differences")
    e = 2.0 ** -7
    for k, t in enumerate((x, r, i, A, h0)):
        d = torch.randn(t.shape, generator=g, device=DEV) * (0.05 if k == 3 else 1.0)
        at = [list((x, r, i, A, h0)) for _ in range(2)]
        at[0][k], at[1][k] = t + e * d, t - e * d
        diff = (loss(run(at[0])) - loss(run(at[1]))) / (2 * e)
        got = float((grads[k].double() * d.double()).sum())
        tol = noise / e + e * e / 6 * 400 * float((grads[k].abs() * d.abs()).sum()) ** 0.5 * 40
        print(f"  {k}: {got:.5f} {diff:.5f} tolerance {tol:.5f}", flush=True)
        assert abs(got - diff) <= tol


@pytest.mark.parametrize("shape", [(0, 5, 8), (2, 0, 8), (0, 0, 8)])
def test_recurrence_nothing(shape):
    announce("nothing", shape)
    b, n, d = shape
    x, r, i = (torch.zeros(shape, device=DEV).requires_grad_() for _ in range(3))
    A = -torch.ones(d, device=DEV).requires_grad_()
    h0 = torch.arange(b * d, device=DEV, dtype=torch.float32).view(b, d).requires_grad_()
    h, last = ops.gated_linear_recurrence(x, r, i, A, h0, None, True)
    assert h.shape == shape and torch.equal(last, h0)
    assert torch.equal(ops.gated_linear_recurrence(x, r, i, A, None, None, True)[1], torch.zeros_like(h0))
    got = torch.autograd.grad((h, last), (x, r, i, h0), (torch.zeros_like(h), torch.ones_like(last)))
    assert torch.equal(got[3], torch.ones_like(h0)) and got[0].shape == shape


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch,dim", [(1, 1), (3, 5), (16, 2560), (64, 333)])
def test_update(batch, dim, dtype):
    """Steps one after the other against the whole row."""
    announce("update", batch, dim, dtype)
    n = 9
    x, r, i, A, h0, _, _, _ = inputs(batch, n, dim, dtype, fused=True, carried=True)
    want = Reference(x, r, i, A, h0, None)
    state, kept = h0.clone(), h0.clone()
    own = h0.clone()
    for t in range(n):
        new, y = ops.gated_linear_recurrence_update(state, x[:, t], r[:, t], i[:, t], A)
        assert new.data_ptr() != state.data_ptr() and y.dtype == x.dtype
        within(y, want.h[:, t], want.eh[:, t] + u(DT[dtype]) * want.h[:, t].abs() + 1e-38, f"step {t}")
        back, y2 = ops.gated_linear_recurrence_update(own, x[:, t], r[:, t], i[:, t], A, inplace=True)
        assert back is own and torch.equal(own, new) and torch.equal(y, y2)
        state = new
    assert torch.equal(h0, kept)
    s16, _ = ops.gated_linear_recurrence_update(h0.bfloat16(), x[:, 0], r[:, 0], i[:, 0], A, inplace=True)
    s32, _ = ops.gated_linear_recurrence_update(h0.bfloat16().float(), x[:, 0], r[:, 0], i[:, 0], A)
    assert s16.dtype == torch.float32 and torch.equal(s16, s32)
    none = ops.gated_linear_recurrence_update(h0[:0], x[:0, 0], r[:0, 0], i[:0, 0], A)
    assert none[0].shape == (0, dim) and none[1].shape == (0, dim)


def test_recurrence_graph_and_streams():
    """Captured forward, gradient and steps give on every replay what eager calls give, with other work in
    between; and on a stream of its own."""
    announce("graph")
    x, r, i, A, h0, seq, go, gl = inputs(2, 333, 70, "bf16", packed=60, carried=True)

    def eager(sets):
        leaves = [t.detach().clone().requires_grad_() for t in sets]
        out = ops.gated_linear_recurrence(*leaves, seq, True)
        return [*out, *torch.autograd.grad(out, leaves, (go, gl))]

    buf = [t.clone().requires_grad_() for t in (x, r, i, A, h0)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            out = ops.gated_linear_recurrence(*buf, seq, True)
            got = torch.autograd.grad(out, buf, (go, gl))
        on_side = [*out, *got]
        del out, got
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(on_side, eager((x, r, i, A, h0))):
        assert torch.equal(p, q)
    del on_side
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.gated_linear_recurrence(*buf, seq, True)
        got = [*out, *torch.autograd.grad(out, buf, (go, gl))]
        state, y = ops.gated_linear_recurrence_update(buf[4].detach(), buf[0].detach()[:, 0], buf[1].detach()[:, 0],
                                                      buf[2].detach()[:, 0], buf[3].detach())
    for k in range(4):
        sets = inputs(2, 333, 70, "bf16", packed=60 + k, carried=True)[:5]
        with torch.no_grad():
            for b, t in zip(buf, sets):
                b.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(got, eager(sets)):
            assert torch.equal(p, q)
        s2, y2 = ops.gated_linear_recurrence_update(sets[4], sets[0][:, 0], sets[1][:, 0], sets[2][:, 0], sets[3])
        assert torch.equal(state, s2) and torch.equal(y, y2)


def test_recurrence_long_rows():
    """Offsets past 32 bits: positions that lie more than 2^32 elements apart."""
    announce("long rows")
    stride = 2 ** 29 + 8
    base = torch.zeros(9 * stride + 64, dtype=torch.bfloat16, device=DEV)
    x = base.as_strided((1, 10, 16), (0, stride, 1))
    g = gen("long")
    vals = [torch.randn((1, 10, 16), generator=g, device=DEV).bfloat16() for _ in range(3)]
    x.copy_(vals[0])
    A = -torch.rand(16, generator=g, device=DEV)
    assert torch.equal(ops.gated_linear_recurrence(x, vals[1], vals[2], A),
                       ops.gated_linear_recurrence(vals[0], vals[1], vals[2], A))
