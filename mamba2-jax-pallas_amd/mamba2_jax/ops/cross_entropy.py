"""Softmax cross entropy of a linear head over a vocabulary on MI355X, without the
logits, as HIP kernels in libm2ssd.so (m2_linear_cross_entropy,
m2_linear_cross_entropy_grad).

No counterpart operator in the reference, whose models answer with logits
(models/mamba2_lm.py:213-216): float32 logits of 8192 tokens over a vocabulary of 50288
take 1.6 GB, and their softmax and gradient as much again; here a tile of logits exists
in registers only, forward and backward.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _lib as L
from .embedding import _dense, _rows, _stride

REDUCTIONS = ("mean", "sum", "none")


def _forward(x, weight, targets, ignore_index, reduction, save):
    """-> (the reduction, or the per-position losses; what the gradient reads, or None)"""
    dev, dim = x.device, x.shape[-1]
    xr, w, t = _rows(x, dim), _rows(weight, dim), _dense(targets)
    none = reduction == "none"
    out = torch.empty(targets.shape if none else (), dtype=torch.float32, device=dev)
    args = L.LinearCrossEntropyArgs(
        xr.data_ptr(), w.data_ptr(), t.data_ptr(), out.data_ptr() if none else 0, 0,
        0 if none else out.data_ptr(), t.numel(), w.shape[0], dim, _stride(xr, dim),
        _stride(w, dim), ignore_index, L.dtype_code(w, "weight"), L.index_code(t, "targets"),
        int(reduction == "mean"))
    if none and not t.numel():
        return out, None
    saved = None
    if save:
        size = L.size_of("m2_linear_cross_entropy_saved_size", args)
        saved = torch.empty(size, dtype=torch.uint8, device=dev)
        args.saved, args.saved_bytes = saved.data_ptr(), size
    L.call_with_workspace("m2_linear_cross_entropy", args, dev)
    return out, saved


def _backward(ctx, grad):
    weight, saved = ctx.saved_tensors
    shape, n, ignore_index, reduction, index_code, weight_shape, dtype, size = ctx.args
    # (hooks may have given them back at other places and strides)
    L.device_of(weight, saved)
    L.require_saved(weight, weight_shape, dtype, "weight")
    want_x, want_w = ctx.needs_input_grad[:2]
    dev, dim = weight.device, weight.shape[1]
    dx = weight.new_empty(shape) if want_x else None
    dw = weight.new_empty(weight.shape) if want_w else None
    if n == 0:
        return dx, None if dw is None else dw.zero_(), None, None, None
    L.require_saved(saved, (size,), torch.uint8, "the loss's kept rows")
    w, saved = _rows(weight, dim), L.dev_contig(saved)
    g = grad.reshape(-1) if grad.dim() != 1 else grad
    if g.dtype != torch.float32:
        g = g.float()
    args = L.LinearCrossEntropyGradArgs(
        0, w.data_ptr(), 0, 0, 0, g.data_ptr(), L.ptr(dx), L.ptr(dw), n, w.shape[0], dim, dim,
        _stride(w, dim), ignore_index, 0 if reduction != "none" else g.stride(0),
        L.dtype_code(w, "weight"), index_code, int(reduction == "mean"))
    args.saved, args.saved_bytes = saved.data_ptr(), saved.numel()
    L.call_with_workspace("m2_linear_cross_entropy_grad", args, dev)
    return dx, dw, None, None, None


_backward_once = once_differentiable(_backward)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, ignore_index, reduction):
        out, saved = _forward(x, weight, targets, ignore_index, reduction, True)
        # (x is not read again: its kept rows are in `saved`)
        ctx.save_for_backward(weight, saved)
        ctx.args = (x.shape, targets.numel(), ignore_index, reduction, L.index_code(targets, "targets"), weight.shape,
                    weight.dtype, 0 if saved is None else saved.numel())
        return out

    @staticmethod
    def backward(ctx, grad):
        # (once_differentiable's own bookkeeping only where a second derivative is recorded)
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, grad)


def linear_cross_entropy(x, weight, targets, ignore_index=-100, reduction="mean"):
    """Cross entropy of softmax(x @ weight.T) against targets, float32; differentiable
    in x and weight.

    x (..., dim) and weight (vocab, dim), both bfloat16 or both float32, rows with a
    contiguous last dimension read in place; targets (...) int32 or int64.
    Positions with targets == ignore_index are left out: their loss and their
    gradient are 0, and what x holds there (a NaN, say) reaches nothing.  A target outside the
    vocabulary cannot be reported without waiting for the GPU: its loss is NaN.

    reduction: "mean" (over the positions kept; 0 where there are none) and "sum"
    return a scalar, "none" the per-position losses in targets' shape.  Sums, the softmax's
    maximum and sum and the loss are float32 or wider.  A logit of +inf or NaN makes
    its loss and gradients NaN; a target's of -inf has loss inf and the
    gradient of softmax - onehot.  The gradient computes the logits again, 512 MB of their
    gradient at a time (or 256 rows of the vocabulary for all tokens, where that is more: a million
    tokens in bfloat16): bfloat16 operands round it to bfloat16 before its products with weight
    and x (float32 sums, each result rounded once), and what that takes from the
    targets' is added in float32, through a float32 row for each token; float32 operands are
    multiplied as three bfloat16 parts each, accurate to about 2^-24 of each product (an
    infinity among them gives NaN).  Between the two the
    graph holds what the kernels read: a packed copy of x's kept rows, and of weight
    where it cannot be read in place (float32, as three bfloat16 parts: 1.5 times
    weight; a dim that 64 does not divide)."""
    L.device_of_two(x, weight)
    L.device_of_two(x, targets)
    shape = x.shape
    L.require(reduction in REDUCTIONS, lambda: f"reduction={reduction!r}: one of {REDUCTIONS}")
    L.require(weight.dim() == 2 and shape and shape[-1] == weight.shape[1],
              lambda: f"x.shape={tuple(shape)}, weight.shape={tuple(weight.shape)}: expected "
                      "(..., dim) and (vocab, dim)")
    L.require(targets.shape == shape[:-1],
              lambda: f"targets.shape={tuple(targets.shape)}: expected {tuple(shape[:-1])}")
    L.require(weight.shape[0] > 0 and weight.shape[1] > 0, lambda: f"weight.shape={tuple(weight.shape)}")
    L.index_code(targets, "targets")
    if L.dtype_code(x, "x") != L.dtype_code(weight, "weight"):
        raise TypeError(f"x is {x.dtype} and weight {weight.dtype}: they must be the same")
    ignore_index = int(ignore_index)
    if (x.requires_grad or weight.requires_grad) and torch.is_grad_enabled():
        return _LinearCrossEntropy.apply(x, weight, targets, ignore_index, reduction)
    L.refuse_tangents(x, weight)
    return _forward(x, weight, targets, ignore_index, reduction, False)[0]


__all__ = ["linear_cross_entropy"]
