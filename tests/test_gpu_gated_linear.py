"""The gated feed-forward product and its gradient against the formulas in 64 bits.

Tolerances are per element and derived from the arithmetic; F = 2^-24, u(T) half a step of T.

* A matrix product over K is off by (K / 4 + 24) F sum |a b| (an instruction adds 32 products in at most
  eight roundings; up to eight partial sums and 64 parts are joined); float32 operands run six such
  sums and leave out 4 F.
* act(g) = g sigmoid(u): u rounds four times, the sigmoid is off by (6 + 2 |u|) F of itself, and
  act's slope is at most 1.13, its second derivative at most 1 in magnitude.
* The gradient reads g and v as they were stored (u(T) of each) and its dg and dv are rounded once more
  (bf16) or split in three parts (4 F).
* What is stored is off by u(T) of itself.
"""

import math
import zlib

import pytest
import torch
import torch.utils.checkpoint

from gpu_util import announce
from mamba2_jax import ops

pytestmark = pytest.mark.gpu

F = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
DEV = "cuda"
C, K3 = math.sqrt(2 / math.pi), 0.044715


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


def product(k, dtype):
    return ((k / 4 + 24) * (6 if dtype == torch.float32 else 1) + (4 if dtype == torch.float32 else 0)) * F


def act(g, activation):
    """(act, its slope, |u|)"""
    if activation == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s), g.abs()
    w = 2 * C * (g + K3 * g ** 3)
    s = torch.sigmoid(w)
    return g * s, s + g * s * (1 - s) * 2 * C * (1 + 3 * K3 * g * g), w.abs()


class Reference:
    def __init__(self, x, w, activation, dh=None):
        dt = x.dtype
        x, w = x.detach().double().reshape(-1, x.shape[-1]), w.detach().double()
        n, d = x.shape
        f = w.shape[0] // 2
        z = x @ w.t()
        ez = product(d, dt) * (x.abs() @ w.abs().t())
        (g, v), (eg, ev) = z.chunk(2, 1), ez.chunk(2, 1)
        a, slope, au = act(g, activation)
        own = (12 + 4 * au.clamp(max=200)) * F
        ea = 1.13 * eg + a.abs() * own
        self.h = a * v
        self.eh = ea * v.abs() + a.abs() * ev + ea * ev + 2 * F * self.h.abs() + u(dt) * self.h.abs() + 1e-37
        if dh is None:
            return
        dh = dh.detach().double().reshape(-1, f)
        ud = u(dt) if dt == torch.bfloat16 else 4 * F
        eg, ev = eg + u(dt) * g.abs(), ev + u(dt) * v.abs()
        dv, dg = dh * a, dh * v * slope
        edv = dh.abs() * (1.13 * eg + a.abs() * own) + (ud + 2 * F) * dv.abs()
        eslope = eg + (1 + g.abs().clamp(max=10)) * 2 * own
        edg = dh.abs() * (slope.abs() * ev + (v.abs() + ev) * eslope) + (ud + 4 * F) * dg.abs()
        dz, edz = torch.cat([dg, dv], 1), torch.cat([edg, edv], 1)
        self.dx = dz @ w
        self.edx = edz @ w.abs() + product(2 * f, dt) * (dz.abs() @ w.abs()) + u(dt) * self.dx.abs() + 1e-37
        self.dw = dz.t().contiguous() @ x
        self.edw = (edz.t().contiguous() @ x.abs() + product(n, dt) * (dz.abs().t().contiguous() @ x.abs())
                    + u(dt) * self.dw.abs() + 1e-37)


def inputs(n, dim, hidden, dtype, scale=1.0):
    g = gen("glu", n, dim, hidden)
    dt = DT[dtype]
    x = torch.randn((n, dim), generator=g, device=DEV).to(dt)
    w = (torch.randn((2 * hidden, dim), generator=g, device=DEV) * (scale / math.sqrt(dim))).to(dt)
    dh = torch.randn((n, hidden), generator=g, device=DEV).to(dt)
    return x, w, dh


def check(x, w, dh, activation):
    want = Reference(x, w, activation, dh)
    with torch.no_grad():
        h = ops.gated_linear(x, w, activation)
    assert h.dtype == x.dtype and h.is_contiguous()
    within(h.reshape(want.h.shape), want.h, want.eh, "h")
    xl, wl = x.detach().requires_grad_(), w.detach().requires_grad_()
    h2 = ops.gated_linear(xl, wl, activation)
    assert torch.equal(h, h2)
    dx, dw = torch.autograd.grad(h2, (xl, wl), dh, retain_graph=True)
    within(dx.reshape(want.dx.shape), want.dx, want.edx, "dx")
    within(dw, want.dw, want.edw, "dw")
    one = torch.autograd.grad(h2, (xl,), dh, retain_graph=True) + torch.autograd.grad(h2, (wl,), dh)
    assert torch.equal(one[0], dx) and torch.equal(one[1], dw)
    return h, dx, dw


SIZES = [(1, 1, 1), (1, 8, 1), (2, 16, 3), (1, 64, 64), (5, 33, 7), (16, 128, 20), (17, 24, 129), (33, 256, 8), (64, 136, 65),
         (64, 1001, 30), (65, 64, 64), (100, 300, 500), (70, 72, 1), (130, 1, 33), (333, 1001, 1365), (257, 192, 128)]


@pytest.mark.parametrize("n,dim,hidden", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_gated_linear(n, dim, hidden, dtype, activation):
    announce("gated linear", n, dim, hidden, dtype, activation)
    check(*inputs(n, dim, hidden, dtype), activation)


# whole rounds of tiles and cut ones; both halves in place and packed
LARGE = [(2000, 512, 1000), (4096, 256, 640), (1024, 768, 2048), (300, 2560, 6912), (3000, 640, 4224), (16, 2560, 6912),
         (48, 2048, 1024)]


@pytest.mark.parametrize("n,dim,hidden", LARGE)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gated_linear_large(n, dim, hidden, dtype):
    announce("gated linear large", n, dim, hidden, dtype)
    check(*inputs(n, dim, hidden, dtype), "silu")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("n", [3, 100])
def test_gated_linear_far_gates(n, dtype, activation):
    """Gates far out on both sides, where the sigmoid ends: no inf - inf, no 0 inf."""
    announce("far gates", n, dtype, activation)
    x, w, dh = inputs(n, 64, 64, dtype, scale=40.0)
    check(x, w, dh, activation)
    # beyond what the exponential takes: act is g or 0, its slope 1 or 0
    x, w, dh = torch.zeros_like(x), torch.zeros_like(w), dh
    x[:, 0], x[:, 1] = 2.0 ** 40, 1.0
    for k in range(64):
        w[k, 0] = (-1.0) ** k * 2.0 ** (k // 4)
        w[64 + k, 1] = 1.0
    h, dx, dw = check(x, w, dh, activation)
    assert torch.equal(h[:, 1::2], torch.zeros_like(h[:, 1::2])) and bool((h[:, 0::2] > 1e12).all())


def test_gated_linear_not_numbers():
    """A NaN or an infinity in a token's row reaches that token's results, and what sums over tokens; one in
    a weight's row the place it makes."""
    announce("not numbers")
    for n in (5, 200):
        x, w, dh = inputs(n, 64, 64, "bf16")
        x[2, 5] = float("nan")
        h, dx, _ = [t.detach() for t in grads(x, w, dh)]
        assert bool(h[2].isnan().all()) and bool(dx[2].isnan().all())
        rest = [k for k in range(n) if k != 2]
        assert bool(h[rest].isfinite().all()) and bool(dx[rest].isfinite().all())
        x, w, dh = inputs(n, 64, 64, "bf16")
        w[7, 3] = float("nan")
        h = ops.gated_linear(x, w)
        assert bool(h[:, 7].isnan().all()) and bool(h[:, [k for k in range(64) if k != 7]].isfinite().all())


def grads(x, w, dh, activation="silu"):
    xl, wl = x.detach().requires_grad_(), w.detach().requires_grad_()
    h = ops.gated_linear(xl, wl, activation)
    return [h, *torch.autograd.grad(h, (xl, wl), dh)]


@pytest.mark.parametrize("n,dim,hidden", [(7, 64, 48), (40, 136, 100), (150, 128, 64), (90, 200, 77)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gated_linear_layouts(n, dim, hidden, dtype):
    """Views of every stride and alignment against the same values laid out plainly: where the
    operands are read in place or packed the sums may be cut differently, so within both tolerances."""
    announce("layouts", n, dim, hidden, dtype)
    x, w, dh = inputs(n, dim, hidden, dtype)
    want = Reference(x, w, "silu", dh)
    wide = torch.full((n, dim + 9), float("nan"), device=DEV, dtype=x.dtype)
    wide[:, 3:3 + dim] = x
    ww = torch.full((2 * hidden, dim + 16), float("nan"), device=DEV, dtype=x.dtype)
    ww[:, 8:8 + dim] = w
    odd = torch.empty(2 * hidden * dim + 1, device=DEV, dtype=x.dtype)[1:].view(2 * hidden, dim)
    odd.copy_(w)
    gw = torch.zeros((n, hidden + 5), device=DEV, dtype=x.dtype)
    gw[:, 1:1 + hidden] = dh
    turned = lambda t: t.t().contiguous().t()
    for x2 in (wide[:, 3:3 + dim], turned(x), x):
        for w2 in (ww[:, 8:8 + dim], odd, turned(w)):
            h, dx, dw = grads(x2, w2, gw[:, 1:1 + hidden])
            within(h, want.h, want.eh, "h")
            within(dx, want.dx, want.edx, "dx")
            within(dw, want.dw, want.edw, "dw")
    # more dimensions, a broadcast token and a gradient that all places share
    x3 = x[:6].reshape(2, 3, dim) if n >= 6 else x
    h3 = ops.gated_linear(x3, w)
    assert h3.shape == (2, 3, hidden)
    within(h3.reshape(6, hidden), want.h[:6], want.eh[:6], "three dimensions")
    he = ops.gated_linear(x[:1].expand(n, dim), w)
    assert bool((he == he[:1]).all())
    xl = x.detach().requires_grad_()
    (p,) = torch.autograd.grad(ops.gated_linear(xl, w).sum(), xl)
    (q,) = torch.autograd.grad(ops.gated_linear(xl, w), xl, torch.ones_like(dh))
    assert torch.equal(p, q)
    assert torch.equal(ops.gated_linear(x[0], w), ops.gated_linear(x[:1], w)[0])


@pytest.mark.parametrize("n,dim,hidden", [(40, 64, 64), (128, 128, 64), (90, 200, 77)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gated_linear_saved_elsewhere(n, dim, hidden, dtype):
    """The graph's tensors put away and brought back at other places, strides and alignments (as hooks that keep them in host
    memory do), and a pass that is computed again."""
    announce("saved elsewhere", n, dim, hidden, dtype)
    x, w, dh = inputs(n, dim, hidden, dtype)
    want = Reference(x, w, "silu", dh)

    def odd(t):
        b = torch.empty((t.shape[0], t.shape[1] + 3), device=DEV, dtype=t.dtype)[:, 1:1 + t.shape[1]]
        b.copy_(t.detach())
        return b

    bring = {"plain": lambda t: t.clone(), "odd": lambda t: odd(t) if t.dim() == 2 else t.clone()}
    for x2 in (x, odd(x)):
        for w2 in (w, odd(w)):
            for name, unpack in bring.items():
                xl, wl = x2.detach().requires_grad_(), w2.detach().requires_grad_()
                with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                    h = ops.gated_linear(xl, wl)
                dx, dw = torch.autograd.grad(h, (xl, wl), dh)
                within(dx, want.dx, want.edx, f"dx {name}")
                within(dw, want.dw, want.edw, f"dw {name}")
    xl, wl = x.detach().requires_grad_(), w.detach().requires_grad_()
    with torch.autograd.graph.save_on_cpu():
        h = ops.gated_linear(xl, wl)
    moved = torch.autograd.grad(h, (xl, wl), dh)
    again = torch.utils.checkpoint.checkpoint(ops.gated_linear, xl, wl, use_reentrant=False)
    again = torch.autograd.grad(again, (xl, wl), dh)
    for p, q, r in zip(moved, again, grads(x, w, dh)[1:]):
        assert torch.equal(p, r) and torch.equal(q, r)


def test_gated_linear_nothing():
    announce("nothing")
    x = torch.zeros((0, 64), device=DEV, dtype=torch.bfloat16).requires_grad_()
    w = torch.ones((20, 64), device=DEV, dtype=torch.bfloat16).requires_grad_()
    h = ops.gated_linear(x, w)
    assert h.shape == (0, 10)
    dx, dw = torch.autograd.grad(h, (x, w), torch.zeros_like(h))
    assert dx.shape == (0, 64) and dw.shape == w.shape and not bool(dw.any())
    assert ops.gated_linear(torch.zeros((3, 0, 64), device=DEV, dtype=torch.bfloat16), w.detach()).shape == (3, 0, 10)


def test_gated_linear_differences():
    """The gradients against differences of the operator along random directions: a central difference of
    step e is off by e^2 / 6 of the third derivative and by the products' errors over e."""
    announce("differences")
    for activation in ("silu", "gelu"):
        x, w, dh = inputs(90, 48, 40, "f32")
        _, dx, dw = grads(x, w, dh, activation)
        noise = float((Reference(x, w, activation, dh).eh * dh.double().abs()).sum())
        g = gen("differences", activation)
        e = 2.0 ** -7
        loss = lambda a, b: float((ops.gated_linear(a, b, activation).double() * dh.double()).sum())
        for k in range(2):
            d = torch.randn((x, w)[k].shape, generator=g, device=DEV) * (1.0 if k == 0 else 1 / math.sqrt(48))
            diff = (loss(x + e * d, w) - loss(x - e * d, w)) if k == 0 else (loss(x, w + e * d) - loss(x, w - e * d))
            diff /= 2 * e
            got = float(((dx, dw)[k].double() * d.double()).sum())
            # along d both products move by a normal number of deviation one: third derivatives of order
            # 10 for each of 3600 places, of random signs
            tol = noise / e + e * e / 6 * 10 * 60 * float(dh.abs().max())
            print(f"  {activation} {k}: {got:.5f} {diff:.5f} tolerance {tol:.5f}", flush=True)
            assert abs(got - diff) <= tol


@pytest.mark.parametrize("n", [4, 300])
def test_gated_linear_graph_and_streams(n):
    """Captured, each replay gives what eager calls give, with other work in between; and so does a
    stream of its own."""
    announce("graph", n)
    x, w, dh = inputs(n, 320, 200, "bf16")
    buf = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    run = lambda: (lambda h: [h, *torch.autograd.grad(h, buf, dh)])(ops.gated_linear(*buf))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = [t.detach() for t in run()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(on_side, grads(x, w, dh)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for k in range(4):
        g = gen("replay", k)
        x2 = torch.randn(x.shape, generator=g, device=DEV).bfloat16()
        w2 = (torch.randn(w.shape, generator=g, device=DEV) / 18).bfloat16()
        with torch.no_grad():
            buf[0].copy_(x2)
            buf[1].copy_(w2)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, grads(x2, w2, dh)))


def test_gated_linear_far_rows():
    """Rows of x that lie past 32-bit offsets from each other."""
    announce("far rows")
    stride = 2 ** 29 + 64
    base = torch.zeros(9 * stride + 64, dtype=torch.bfloat16, device=DEV)
    x, w, dh = inputs(10, 64, 64, "bf16")
    far = base.as_strided((10, 64), (stride, 1))
    far.copy_(x)
    want = Reference(x, w, "silu", dh)
    h, dx, dw = grads(far, w, dh)
    within(h, want.h, want.eh, "h")
    within(dx, want.dx, want.edx, "dx")
    within(dw, want.dw, want.edw, "dw")


@pytest.mark.parametrize("n", [3, 70])
def test_gated_linear_wide(n):
    """The largest hidden size but a few: dz's rows lie 2^31 bytes apart within a tile."""
    announce("wide", n)
    x, w, dh = inputs(n, 64, 2 ** 21 - 5, "bf16")
    want = Reference(x, w, "silu", dh)
    h, dx, dw = grads(x, w, dh)
    within(h, want.h, want.eh, "h")
    within(dx, want.dx, want.edx, "dx")
    within(dw, want.dw, want.edw, "dw")
