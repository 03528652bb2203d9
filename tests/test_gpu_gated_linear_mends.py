"""The gated feed-forward product by the norms of its errors, which tell a lost part of an operand that bounds on single
elements let pass, and at sizes past its launches' counts; against the formulas in 64 bits.

F = 2^-24.  Of normal operands, float32:

* A product over K adds up 6 K / 32 instructions' results with up to eight roundings each, at most F of a sum that grows
  as the root of its length: of the result's norm (0.5 sqrt(K) + 1) F at most.  Without one of the three small products (of a high
  and a low part, or of both middle ones) h, dx and dw would be off by 58 to 70 F of their norms (a part's rounding to
  bfloat16 leaves 2^-9.2 of it, so each is about 2^-18.4 of its product's), without all three by 110.
* h = act(g) v: errors of g and v as above reach h with the weights E act'^2 v^2 / E h^2 and 1, 1.44 together of normal g and
  v (of either activation less than 1.5), act itself 6 F.  The factors of the gradient likewise.

bfloat16: what the result is off by is the rounding of dz and its own, both of which the formulas in 64 bits show when
they round at the same two places.  Factors cut to 24 bits (2^-15) add nothing to that; of 16 bits they would add a
quarter.
"""

import math

import pytest
import torch

from gpu_util import announce
from mamba2_jax import ops
from test_gpu_gated_linear import DEV, F, Reference, act, grads, inputs

pytestmark = pytest.mark.gpu


def formula(x, w, dh, activation, rounded=lambda t: t):
    """(h, dx, dw) in 64 bits, dz and the results rounded by `rounded`"""
    x, w, dh = (t.detach().double() for t in (x, w, dh))
    g, v = (x @ w.t()).chunk(2, 1)
    a, slope, _ = act(g, activation)
    dz = rounded(torch.cat([dh * v * slope, dh * a], 1))
    return rounded(a * v), rounded(dz @ w), rounded(dz.t().contiguous() @ x)


def off(got, want):
    return float((got.detach().double() - want).norm() / want.norm())


# 1 to 64 tokens, then the small, middle and large tiles of the forward product
TILES = [(1, 256, 256), (16, 256, 256), (64, 256, 2048), (64, 264, 40), (333, 250, 365), (2000, 256, 1000), (300, 256, 6912),
         (1500, 256, 256)]


@pytest.mark.parametrize("n,dim,hidden", TILES)
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_float32_products_keep_every_part(n, dim, hidden, activation):
    announce("every part", n, dim, hidden, activation)
    x, w, dh = inputs(n, dim, hidden, "f32")
    want = formula(x, w, dh, activation)
    product = lambda k: (0.5 * math.sqrt(k) + 1) * F
    h = 1.5 * product(dim) + 6 * F
    for name, got, ref, tol in zip(("h", "dx", "dw"), grads(x, w, dh, activation), want,
                                   (h, h + product(2 * hidden), h + product(n))):
        e = off(got, ref)
        print(f"  {name}: {e / F:.2f} F of {tol / F:.2f} F", flush=True)
        assert e <= tol, name


@pytest.mark.parametrize("n,dim,hidden", [(16, 512, 700), (64, 256, 2048), (333, 1001, 1365), (2000, 512, 1000), (300, 2560, 6912),
                                          (3000, 640, 1024)])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_bfloat16_gradient_is_off_by_its_two_roundings(n, dim, hidden, activation):
    announce("two roundings", n, dim, hidden, activation)
    x, w, dh = inputs(n, dim, hidden, "bf16")
    want = formula(x, w, dh, activation)
    model = formula(x, w, dh, activation, lambda t: t.bfloat16().double())
    for name, got, ref, m in zip(("h", "dx", "dw"), grads(x, w, dh, activation), want, model):
        e, by = off(got, ref), off(m, ref)
        print(f"  {name}: {e:.3e}, by the roundings {by:.3e}", flush=True)
        assert e <= 1.08 * by, name


def test_more_rows_than_a_launch_counts():
    """Packing of more tokens than 2^32 threads would take a wavefront each."""
    announce("many rows")
    n = 2 ** 26 + 5
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn((n, 1), generator=g, device=DEV).bfloat16()
    w = torch.tensor([[0.75], [-1.5]], device=DEV).bfloat16()
    h = ops.gated_linear(x, w)
    for part in (slice(0, 1000), slice(2 ** 25 - 500, 2 ** 25 + 500), slice(n - 1000, n)):
        t = x[part].double()
        want = 0.75 * t * torch.sigmoid(0.75 * t) * (-1.5 * t)
        assert bool(((h[part].double() - want).abs() <= (2.0 ** -8 + 40 * F) * want.abs() + 1e-37).all())


@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_gated_linear_differences_by_the_formula(activation):
    """The gradients against differences of the operator: what a central difference of step e is off by is taken from
    the formula in 64 bits at the same points, and the products' errors over e from their bounds."""
    announce("differences by the formula", activation)
    x, w, dh = inputs(90, 48, 40, "f32")
    want = Reference(x, w, activation, dh)
    got = grads(x, w, dh, activation)[1:]
    g = torch.Generator(device=DEV).manual_seed(11)
    e = 2.0 ** -4
    up = dh.double()
    for k, name in enumerate(("dx", "dw")):
        t = (x, w)[k]
        d = torch.randn(t.shape, generator=g, device=DEV) * (1.0 if k == 0 else 1 / math.sqrt(48))
        at = [[x, w] for _ in range(2)]
        at[0][k], at[1][k] = t + e * d, t - e * d
        refs = [Reference(*p, activation) for p in at]
        step = (at[0][k].double() - at[1][k].double()) / (2 * e)              # (as float32 has it)
        exact = float(((refs[0].h - refs[1].h) * up).sum()) / (2 * e)
        slope = float((getattr(want, name) * step).sum())
        noise = sum(float((r.eh * up.abs()).sum()) for r in refs) / (2 * e)
        own = float((getattr(want, "e" + name) * step.abs()).sum())
        one = [ops.gated_linear(*p, activation).double() for p in at]
        diff = float(((one[0] - one[1]) * up).sum()) / (2 * e)
        mine = float((got[k].double() * step).sum())
        tol = noise + own + abs(exact - slope)
        print(f"  {name}: {mine:.5f} {diff:.5f} tolerance {tol:.2e}, of it the difference's own {abs(exact - slope):.2e}", flush=True)
        assert abs(mine - diff) <= tol
        assert tol < 0.05 * float((getattr(want, name).abs() * step.abs()).sum())
