"""The gated linear recurrence where its arithmetic ends: infinite states, decays that leave nothing of a large state,
padding around them, offsets past 32 bits; against the formulas in 64 bits.

Tolerances are per element and derived from the arithmetic; F = 2^-24, u(T) half a step of T.

* A gate is off by (6 + 2 |r|) F of itself, L = A q by F more.
* a: where L is below -0.5 it is an exponential, off by |L| (L's own error and 2 F of its product) and 3 F of itself
  (and 2^-126 flushed); above, alpha = 1 - a is off by L's error and 12 F of itself, a by as much of alpha.
  (Between -0.5 and -0.5001 either form may be taken, of which the second allows more.)
* beta = sqrt(1 - a^2), by half of what 1 - a^2 is off by, and 5 F.
* A step rounds what it multiplies and adds at their own sizes: 6 F (a |h| + |b|), a being at least 0.6 where
  h itself is added to b first.  So a state's error decays as the state does, and the error obeys the
  recurrence itself, run here on magnitudes; the joins of maps add 24 F of the sum of the magnitudes.
* A gradient is a product: its factors' errors, times the other factors' magnitudes.
"""

import math

import pytest
import torch

from gpu_util import announce
from mamba2_jax import ops
from mamba2_jax.ops import gated_recurrence as R
from test_gpu_gated_recurrence import DEV, DT, F, gen, inputs, scan, u, within

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


class Sharp:
    """Results in 64 bits, and what a kernel may be off by that keeps the bits of every decay."""

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
        eL = eq + F
        ea = torch.exp(la)
        alpha, y = -torch.expm1(la), -torch.expm1(2 * la)
        far = la < -0.5001
        aerr = torch.where(far, ea * (la.abs() * (eL + 2 * F) + 3 * F) + 2.0 ** -126, alpha * (eL + 12 * F) + F * alpha)
        beta = torch.sqrt(y)
        eb = torch.where(far, (2 * ea * aerr + F) / y.clamp_min(0.5) / 2, 0.65 * (eL + 12 * F)) + 5 * F
        add = torch.where(live, beta * s * x, zero)
        a = torch.where(clear, zero, torch.where(live, ea, zero + 1))
        aerr_h = torch.where(live & ~clear, aerr, zero)          # of what the state is multiplied by
        eadd = (eb + es + 2 * F) * add.abs()
        h0 = zero[:, 0] if h0 is None else h0.detach().double()
        first = lambda t, v: torch.cat([t[:, :1] + a[:, :1] * v[:, None], t[:, 1:]], 1)
        before = lambda t, v: torch.where(clear, zero, torch.cat([v[:, None], t[:, :-1]], 1))
        h = scan(a, first(add, h0))
        mag = scan(a, first(add.abs(), h0.abs()))
        mb = before(mag, h0.abs())
        eh = scan(a, aerr_h * mb + eadd + 6 * F * (a * mb + add.abs())) + 24 * F * mag
        self.h, self.last = torch.where(live, h, zero), h[:, -1]
        self.eh, self.elast = torch.where(live, eh, zero), eh[:, -1]
        if g is None:
            return
        g = torch.where(live, g.detach().double(), zero)
        gl = torch.zeros_like(g[:, 0]) if glast is None else glast.detach().double()
        gmag = torch.cat([g[:, :-1].abs(), g[:, -1:].abs() + gl.abs()[:, None]], 1)
        g = torch.cat([g[:, :-1], g[:, -1:] + gl[:, None]], 1)
        later = torch.cat([a[:, 1:], zero[:, :1]], 1)
        lam = scan(later.flip(1), g.flip(1)).flip(1)
        lmag = scan(later.flip(1), gmag.flip(1)).flip(1)
        passed = aerr_h * lmag + 4 * F * a * lmag
        el = scan(later.flip(1), (torch.cat([passed[:, 1:], zero[:, :1]], 1) + 2 * F * lmag).flip(1)).flip(1) + 24 * F * lmag
        self.dh0 = a[:, 0] * lam[:, 0]
        self.edh0 = (a * el + passed)[:, 0]
        lam, lmag, el = (torch.where(live, t, zero) for t in (lam, lmag, el))
        p, ep = before(h, h0), before(eh, zero[:, 0])
        rise = ea * ea / beta.clamp_min(1e-300) * s * x
        self.dx = lam * beta * s
        self.edx = el * beta * s + lmag * beta * s * (eb + es + 3 * F)
        self.di = self.dx * x * (1 - s)
        self.edi = (self.edx + lmag * beta * s * (2 * es + 5 * F)) * x.abs() * (1 - s)
        dL = lam * (ea * p - rise)
        edL = el * (ea * p - rise).abs() + lmag * (
            ea * ep + aerr * mb + rise.abs() * (2 * aerr / ea.clamp_min(1e-300) + eb + es + 8 * F)
            + 4 * F * (ea * mb + rise.abs()))
        edL = torch.where(live, edL, zero)
        slope = (la * (1 - q)).abs()
        self.dr, self.edr = dL * la * (1 - q), (edL + dL.abs() * (3 * eq + 6 * F)) * slope
        self.dr, self.edr = (torch.where(live, t, zero) for t in (self.dr, self.edr))
        terms = torch.where(live, dL * q, zero)
        self.dA = terms.sum((0, 1))
        self.edA = (edL * q + terms.abs() * (eq + 2 * F)).sum((0, 1)) + b * n * F * terms.abs().sum((0, 1))


def spikes(t, g, big):
    """Every tenth entry or so `big` times the others."""
    return torch.where(torch.rand(t.shape, generator=g, device=DEV) < 0.1, t * big, t)


def sharp_check(x, r, i, A, h0, seq, go, gl):
    want = Sharp(x, r, i, A, h0, seq, go, gl)
    leaves = [t.detach().clone().requires_grad_() for t in (x, r, i, A, h0)]
    h, last = ops.gated_linear_recurrence(*leaves, seq, True)
    within(h, want.h, want.eh + u(h.dtype) * want.h.abs() * (h.dtype == torch.bfloat16) + 1e-37, "h")
    within(last, want.last, want.elast + 1e-37, "last")
    for name, got in zip(("dx", "dr", "di", "dA", "dh0"), torch.autograd.grad((h, last), leaves, (go, gl))):
        ref = getattr(want, name)
        tol = getattr(want, "e" + name) + (u(got.dtype) * ref.abs() if got.dtype == torch.bfloat16 else 0) + 1e-36
        within(got, ref, tol, name)


# from decays that no step takes below -0.5 to ones that leave nothing, and all of them in neighbouring channels
DECAYS = [(0.3, 2.0), (16.0, 60.0), (1e-3, 200.0)]


# (the last of the sizes: rows whose backward passes segments on)
STRONG = [(*size, *decay) for size in [(2, 300, 40, 0), (1, 1100, 70, 0), (3, 333, 65, 40)] for decay in DECAYS] + [
    (9, 1100, 3713, 0, 16.0, 60.0)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("batch,seqlen,dim,packed,low,high", STRONG)
def test_recurrence_keeps_small_inputs_behind_large_states(batch, seqlen, dim, packed, dtype, low, high):
    """What a strong decay leaves of a state, however large, does not round what comes in, forward or backward."""
    announce("strong decay", batch, seqlen, dim, packed, dtype, low, high)
    x, r, i, A, h0, seq, go, gl = inputs(batch, seqlen, dim, dtype, packed=packed, carried=True, low=low, high=high)
    g = gen("spikes", batch, seqlen, dim, low)
    x, go = (spikes(t * 2.0 ** -10, g, 2.0 ** 24) for t in (x, go))
    sharp_check(x, r, i, A, h0 * 2.0 ** 20, seq, go, gl * 2.0 ** 20)


@pytest.mark.parametrize("low,high", DECAYS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_update_keeps_small_inputs_behind_large_states(dtype, low, high):
    announce("strong decay, steps", dtype, low, high)
    x, r, i, A, h0, _, _, _ = inputs(3, 12, 70, dtype, fused=True, carried=True, low=low, high=high)
    x, h0 = x * 2.0 ** -10, h0 * 2.0 ** 20
    want = Sharp(x, r, i, A, h0, None)
    state = h0
    for t in range(12):
        state, y = ops.gated_linear_recurrence_update(state, x[:, t], r[:, t], i[:, t], A)
        tol = want.eh[:, t] + 1e-37
        within(state, want.h[:, t], tol, f"state {t}")
        within(y, want.h[:, t], tol + u(y.dtype) * want.h[:, t].abs(), f"step {t}")


INFINITE = [(*size, decay) for size in [(1, 5, 3), (2, 900, 66)] for decay in (-1e-3, -0.4, -5.0, -40.0, -200.0, -2000.0)] + [
    (9, 1100, 3713, -40.0)]


@pytest.mark.parametrize("batch,seqlen,dim,decay", INFINITE)
def test_recurrence_infinite_states_stay(batch, seqlen, dim, decay):
    """a is never 0: an infinite state, or gradient of one, stays what it is until a sequence ends, and no
    neighbour sees it."""
    announce("infinite states", decay, batch, seqlen, dim)
    x, r, i, A, h0, _, go, gl = inputs(batch, seqlen, dim, "f32", carried=True)
    A = torch.full_like(A, decay)
    bad_h, bad_g, bad_x = h0.clone(), gl.clone(), x.clone()
    bad_h[0, 0], bad_g[0, 1], bad_x[0, 2, 2] = INF, -INF, -INF

    def run(x, h0, gl):
        leaves = [t.clone().requires_grad_() for t in (x, r, i, A, h0)]
        out = ops.gated_linear_recurrence(*leaves, None, True)
        return [t.detach() for t in out], torch.autograd.grad(out, leaves, (go, gl))

    (h, last), _ = run(bad_x, bad_h, gl)
    assert bool((h[0, :, 0] == INF).all()) and float(last[0, 0]) == INF
    assert bool((h[0, 2:, 2] == -INF).all()) and float(last[0, 2]) == -INF
    (clean, clean_last), grads = run(x, h0, gl)
    for p, q in ((h, clean), (last, clean_last)):
        q = q.clone()
        q[0, ..., 0], q[0, ..., 2] = p[0, ..., 0], p[0, ..., 2]
        assert torch.equal(p, q)
    assert torch.equal(h[0, :2, 2], clean[0, :2, 2])
    _, (dx, dr, di, dA, dh0) = run(x, h0, bad_g)
    assert float(dh0[0, 1]) == -INF and bool((dx[0, :, 1] == -INF).all())
    for p, q in zip((dx, dr, di, dA, dh0), grads):
        p, q = p.clone(), q.clone()
        p[..., 1], q[..., 1] = 0, 0
        assert torch.equal(p, q)
    # one token at a time
    state = bad_h
    for t in range(min(seqlen, 12)):
        state, y = ops.gated_linear_recurrence_update(state, bad_x[:, t], r[:, t], i[:, t], A)
        assert torch.equal(state[0, 0], last[0, 0]) and float(y[0, 0]) == INF
    assert float(state[0, 2]) == -INF
    # until a sequence ends
    seq = torch.zeros((batch, seqlen), dtype=torch.int32, device=DEV)
    seq[:, 3:] = 1
    h = ops.gated_linear_recurrence(bad_x, r, i, A, bad_h, seq)
    assert bool((h[0, :3, 0] == INF).all()) and bool(h[:, 3:].isfinite().all())


@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("seqlen", [7, 300])
def test_recurrence_states_that_pass_padding_alone(value, seqlen):
    """A row of padding hands its state on, whatever it is, and takes no part in any gradient but that state's."""
    announce("padding alone", value, seqlen)
    x, r, i, A, h0, _, go, gl = inputs(3, seqlen, 37, "f32", carried=True)
    seq = torch.zeros((3, seqlen), dtype=torch.int32, device=DEV)
    seq[1] = -1
    seq[2, seqlen - 3:] = -1

    def run(h0, gl):
        leaves = [t.clone().requires_grad_() for t in (x, r, i, A, h0)]
        out = ops.gated_linear_recurrence(*leaves, seq, True)
        return [t.detach() for t in out], torch.autograd.grad(out, leaves, (go, gl))

    (h, last), grads = run(h0, gl)
    bad_h, bad_g = h0.clone(), gl.clone()
    bad_h[1, 5], bad_g[1, 9] = value, value
    (h2, last2), grads2 = run(bad_h, bad_g)
    assert torch.equal(h, h2) and torch.equal(last2.view(torch.int32)[1], bad_h.view(torch.int32)[1])
    for name, p, q in zip(("dx", "dr", "di", "dA"), grads, grads2):
        assert torch.equal(p, q), name
    got = grads2[4][1]
    assert bool(((got == bad_g[1]) | (got.isnan() & bad_g[1].isnan())).all())


def test_recurrence_positive_decay():
    """A above 0 is not a decay: NaN in its channel, whatever its neighbours' are."""
    announce("positive A")
    x, r, i, A, h0, _, _, _ = inputs(2, 40, 8, "f32", carried=True)
    for other in (-0.1, -30.0):
        A = torch.full_like(A, other)
        A[3] = 0.2
        h = ops.gated_linear_recurrence(x, r, i, A, h0)
        state, y = ops.gated_linear_recurrence_update(h0, x[:, 0], r[:, 0], i[:, 0], A)
        for t in (h, state[:, None], y[:, None]):
            bad = t.isnan()
            assert bool(bad[..., 3].all()) and not bool(bad[..., [0, 1, 2, 4, 5, 6, 7]].any())


@pytest.mark.parametrize("batch,seqlen,dim,strides", [(3, 40, 16, (2 ** 31 + 8, 16, 1)), (1, 4200, 16, (0, 2 ** 20, 1))])
def test_recurrence_in_place_past_32_bits(batch, seqlen, dim, strides):
    """Views read in place whose rows, or positions, lie more than 2^32 bytes apart, forward and backward."""
    announce("in place past 32 bits", batch, seqlen, dim, strides)
    x, r, i, A, h0, _, go, gl = inputs(batch, seqlen, dim, "bf16", carried=True)
    apart = dim if strides[1] > dim else seqlen * dim + 24           # of the four streams
    base = torch.empty((batch - 1) * strides[0] + (seqlen - 1) * strides[1] + 4 * apart, device=DEV, dtype=torch.bfloat16)
    assert 2 * base.numel() > 2 ** 32
    views = [base.as_strided((batch, seqlen, dim), strides, k * apart).copy_(t) for k, t in enumerate((x, r, i, go))]
    for v in views:
        assert R._strided(v) is v

    def run(x, r, i, go):
        leaves = [t.detach().requires_grad_() for t in (x, r, i)] + [t.clone().requires_grad_() for t in (A, h0)]
        out = ops.gated_linear_recurrence(*leaves, None, True)
        return [*out, *torch.autograd.grad(out, leaves, (go, gl))]

    for p, q in zip(run(*views), run(x, r, i, go)):
        assert torch.equal(p, q)


def test_recurrence_results_past_32_bits():
    """Outputs, the states between them and gradients of more than 2^31 elements: the row's end against a row of its own."""
    announce("results past 32 bits")
    n, d, tail = 2 ** 21 + 261, 1032, 700
    g = gen("huge")
    x, r, i, go = (torch.empty((1, n, d), device=DEV, dtype=torch.bfloat16).normal_(generator=g) for _ in range(4))
    assert x.numel() > 2 ** 31
    A = -torch.rand(d, generator=g, device=DEV) - 1e-3
    seq = torch.zeros((1, n), dtype=torch.int32, device=DEV)
    seq[:, n - tail:] = 1
    leaves = [t.requires_grad_() for t in (x, r, i)]
    h, last = ops.gated_linear_recurrence(*leaves, A, None, seq, True)
    grads = torch.autograd.grad(h, leaves, go)
    cut = [t.detach()[:, n - tail:].contiguous() for t in (x, r, i)]
    want = Sharp(*cut, A, None, None, go[:, n - tail:])
    within(h[:, n - tail:], want.h, want.eh + u(h.dtype) * want.h.abs() + 1e-37, "h")
    within(last, want.last, want.elast + 1e-37, "last")
    for name, got in zip(("dx", "dr", "di"), grads):
        ref = getattr(want, name)
        within(got[:, n - tail:], ref, getattr(want, "e" + name) + u(got.dtype) * ref.abs() + 1e-36, name)


def test_recurrence_differences_by_the_formula():
    """The gradients against differences of the operator: what a central difference of step e is off by is taken
    from the formula in 64 bits at the same points, and the sums' errors over e from their bounds."""
    announce("differences by the formula")
    for low, high in ((0.05, 0.5), (0.2, 6.0)):
        x, r, i, A, h0, seq, go, gl = inputs(2, 120, 9, "f32", packed=50, carried=True, low=low, high=high)
        leaves = [t.clone().requires_grad_() for t in (x, r, i, A, h0)]
        run = lambda ts: ops.gated_linear_recurrence(*ts, seq, True)
        dot = lambda h, last: float((h.double() * go.double()).sum() + (last.double() * gl.double()).sum())
        grads = torch.autograd.grad(run(leaves), leaves, (go, gl))
        want = Sharp(x, r, i, A, h0, seq, go, gl)
        g = gen("differences by the formula", low)
        e = 2.0 ** -4
        for k, name in enumerate(("dx", "dr", "di", "dA", "dh0")):
            t = (x, r, i, A, h0)[k]
            d = torch.randn(t.shape, generator=g, device=DEV)
            if name == "dA":
                d = d * A.abs()
            at = [[*(x, r, i, A, h0)] for _ in range(2)]
            at[0][k], at[1][k] = t + e * d, t - e * d
            refs = [Sharp(*ts, seq) for ts in at]
            step = (at[0][k].double() - at[1][k].double()) / (2 * e)       # (as float32 has it)
            exact = (dot(refs[0].h, refs[0].last) - dot(refs[1].h, refs[1].last)) / (2 * e)
            slope = float((getattr(want, name) * step).sum())
            noise = sum(float((q.eh * go.double().abs()).sum() + (q.elast * gl.double().abs()).sum()) for q in refs)
            diff = (dot(*run(at[0])) - dot(*run(at[1]))) / (2 * e)
            got = float((grads[k].double() * step).sum())
            own = float((getattr(want, "e" + name) * step.abs()).sum())
            tol = noise / (2 * e) + own + abs(exact - slope)
            print(f"  {name}: {got:.6f} {diff:.6f} tolerance {tol:.2e}, of it the difference's own {abs(exact - slope):.2e}", flush=True)
            assert abs(got - diff) <= tol
            assert math.isfinite(tol) and tol < 0.05 * float((getattr(want, name).abs() * step.abs()).sum())


def turned(t):
    """t's values with its last dimension's stride the largest."""
    return t.detach().movedim(-1, 0).contiguous().movedim(0, -1) if t.dim() > 1 else t.detach().clone()


@pytest.mark.parametrize("bring", ["plain", "turned", "odd"])
def test_saved_tensors_elsewhere(bring):
    """What the graphs saved, given back at other places, strides and alignments: the same gradients."""
    announce("saved elsewhere", bring)

    def odd(t):
        b = torch.empty(t.numel() + 1, device=t.device, dtype=t.dtype)[1:].view(t.shape)
        return b.copy_(t.detach())

    unpack = {"plain": lambda t: t.detach().clone(), "turned": turned, "odd": odd}[bring]
    x, r, i, A, h0, seq, go, gl = inputs(2, 150, 24, "bf16", packed=40, carried=True)
    g = gen("saved elsewhere")
    rows, w = (torch.randn(s, generator=g, device=DEV) for s in ((70, 40), (96, 40)))
    up = torch.randn((70, 48), generator=g, device=DEV)
    targets = torch.randint(0, 96, (70,), generator=g, device=DEV)
    calls = [
        (lambda *t: ops.gated_linear_recurrence(*t, seq, True), (x, r, i, A, h0), (go, gl)),
        (lambda *t: ops.gated_linear(*t), (rows, w), (up,)),
        (lambda *t: ops.linear_cross_entropy(*t, targets), (rows, w), (torch.ones((), device=DEV),)),
        (lambda t: ops.embedding(targets, t), (w,), (torch.randn((70, 40), generator=g, device=DEV),)),
    ]
    for fn, args, ups in calls:
        def run(hooks):
            leaves = [t.detach().clone().requires_grad_() for t in args]
            if hooks is None:
                out = fn(*leaves)
            else:
                with hooks:
                    out = fn(*leaves)
            return torch.autograd.grad(out, leaves, ups)

        want = run(None)
        for hooks in (torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack), torch.autograd.graph.save_on_cpu()):
            for p, q in zip(run(hooks), want):
                assert torch.equal(p, q)
