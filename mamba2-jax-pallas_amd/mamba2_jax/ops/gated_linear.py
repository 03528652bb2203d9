"""The first half of a gated feed-forward block on MI355X, h = act(x Wg^T) * (x Wv^T), and its
gradient, as HIP kernels in libm2ssd.so (m2_gated_linear, m2_gated_linear_grad).

No counterpart operator in the reference, whose blocks have a mixer alone
(models/mamba2_lm.py:196-211).  Both products, the activation and the product of the two
are one kernel: neither product is stored unless a gradient asks for it.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _lib as L
from .embedding import _rows, _stride


def _forward(x, weight, activation, save):
    """-> (h, x and weight as they are read, what else the gradient reads or None)"""
    dev, dim = weight.device, weight.shape[1]
    hidden = weight.shape[0] // 2
    xr, w = _rows(x, dim), _rows(weight, dim)
    n = xr.shape[0]
    h = torch.empty((*x.shape[:-1], hidden), dtype=x.dtype, device=dev)
    if n == 0:
        return h, xr, w, None
    args = L.GatedLinearArgs(xr.data_ptr(), w.data_ptr(), h.data_ptr(), n, dim, hidden,
                             _stride(xr, dim), _stride(w, dim), L.dtype_code(w, "weight"), activation)
    saved = None
    if save:
        size = L.size_of("m2_gated_linear_saved_size", args)
        saved = torch.empty(size, dtype=torch.uint8, device=dev)
        args.saved, args.saved_bytes = saved.data_ptr(), size
    L.call_with_workspace("m2_gated_linear", args, dev)
    return h, xr, w, saved


def _backward(ctx, grad):
    xr, w, saved = ctx.saved_tensors
    want_x, want_w = ctx.needs_input_grad[:2]
    x_shape, w_shape, size, dtype = ctx.saved_as
    (n, dim), hidden = x_shape, w_shape[0] // 2
    # (hooks may have given them back at other places and strides)
    at = w.get_device()
    if at < 0 or xr.get_device() != at or (n and saved.get_device() != at):
        L.device_of(xr, w, saved)
    if not (xr.shape == x_shape and w.shape == w_shape and xr.dtype == w.dtype == dtype):
        L.require_saved(xr, x_shape, dtype, "x")
        L.require_saved(w, w_shape, dtype, "weight")
    xr, w = _rows(xr, dim), _rows(w, dim)
    dx = torch.empty(ctx.shape, dtype=w.dtype, device=w.device) if want_x else None
    dw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if want_w else None
    if n == 0:
        return dx, None if dw is None else dw.zero_(), None
    L.require_saved(saved, size, torch.uint8, "the product's factors")
    saved = L.dev_contig(saved)
    g = _rows(grad, hidden)
    args = L.GatedLinearGradArgs(
        xr.data_ptr(), w.data_ptr(), saved.data_ptr(), size[0], g.data_ptr(), L.ptr(dx), L.ptr(dw), n, dim,
        hidden, _stride(xr, dim), _stride(w, dim), _stride(g, hidden), L.dtype_code(w, "weight"),
        ctx.activation)
    L.call_with_workspace("m2_gated_linear_grad", args, w.device)
    return dx, dw, None


_backward_once = once_differentiable(_backward)


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, activation):
        h, xr, w, saved = _forward(x, weight, activation, True)
        # (the rows that were read: the same strides and alignment decide what lies in `saved`)
        ctx.save_for_backward(xr, w, saved)
        ctx.shape, ctx.activation = x.shape, activation
        ctx.saved_as = xr.shape, w.shape, None if saved is None else saved.shape, w.dtype
        return h

    @staticmethod
    def backward(ctx, grad):
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, grad)


def gated_linear(x, weight, activation="silu"):
    """-> act(x @ weight[:hidden].T) * (x @ weight[hidden:].T), shape (..., hidden), x's dtype;
    differentiable in x and weight.

    x (..., dim) and weight (2 hidden, dim), both bfloat16 or both float32, rows with a contiguous
    last dimension read in place: the gate's rows first, then the values'.  activation: "silu", or
    "gelu" in its tanh form.

    Sums and the activation are float32, h is rounded once; float32 operands are multiplied as three
    bfloat16 parts each, accurate to about 2^-24 of each product (an infinity among them gives
    NaN).  Between the two the graph holds x, weight, act(g) and v act'(g) of the two products g and v (for
    bfloat16 operands 24 bits of each), and a packed copy of the operands that the kernels cannot read in
    place (float32, as three bfloat16 parts: 1.5 times each; a dim or hidden that 64 does not divide); the
    gradient of bfloat16 operands rounds its products with those to bfloat16 once.
    Inputs that carry forward-mode derivatives are refused.  Equal inputs give equal bits."""
    dev = L.device_of_two(x, weight)
    shape = x.shape
    L.require(weight.dim() == 2 and shape and shape[-1] == weight.shape[1],
              lambda: f"x.shape={tuple(shape)}, weight.shape={tuple(weight.shape)}: expected "
                      "(..., dim) and (2 hidden, dim)")
    L.require(weight.shape[0] > 0 and weight.shape[0] % 2 == 0 and weight.shape[1] > 0,
              lambda: f"weight.shape={tuple(weight.shape)}: expected (2 hidden, dim)")
    if activation not in L.ACTIVATIONS:
        raise L.M2ShapeError(f"activation={activation!r}: one of {tuple(L.ACTIVATIONS)}")
    if L.dtype_code(x, "x") != L.dtype_code(weight, "weight"):
        raise TypeError(f"x is {x.dtype} and weight {weight.dtype}: they must be the same")
    code = L.ACTIVATIONS[activation]
    if (x.requires_grad or weight.requires_grad) and torch.is_grad_enabled():
        return _GatedLinear.apply(x, weight, code)
    L.refuse_tangents(x, weight)
    return _forward(x, weight, code, False)[0]


__all__ = ["gated_linear"]
