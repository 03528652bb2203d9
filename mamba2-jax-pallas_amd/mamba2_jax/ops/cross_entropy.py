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
from .embedding import _rows, _stride

REDUCTIONS = ("mean", "sum", "none")


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, ignore_index, reduction):
        dev = x.device
        dim = int(x.shape[-1])
        xr, w = _rows(x.detach(), dim), _rows(weight.detach(), dim)
        t = targets.reshape(-1).contiguous()
        n, vocab = t.numel(), int(w.shape[0])
        loss = torch.empty(targets.shape, dtype=torch.float32, device=dev)
        lse = torch.empty_like(loss)
        total = None if reduction == "none" else torch.empty((), dtype=torch.float32, device=dev)
        args = L.LinearCrossEntropyArgs(
            x=L.ptr(xr), weight=L.ptr(w), targets=L.ptr(t), loss=L.ptr(loss), lse=L.ptr(lse),
            total=L.ptr(total), n=n, vocab=vocab, dim=dim, ldx=_stride(xr, dim),
            ldw=_stride(w, dim), ignore_index=int(ignore_index), dtype=L.dtype_code(w, "weight"),
            target_dtype=L.index_code(t, "targets"), mean=int(reduction == "mean"))
        L.call_with_workspace("m2_linear_cross_entropy", args, dev)
        # the per-token losses are the result where nothing is reduced: what the backward
        # reads is then a copy, which the caller's in-place changes do not reach
        kept = loss.clone() if total is None and (ctx.needs_input_grad[0] or ctx.needs_input_grad[1]) \
            else loss
        ctx.save_for_backward(x, weight, t, kept, lse)
        ctx.args = int(ignore_index), reduction
        return loss if total is None else total

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, t, loss, lse = ctx.saved_tensors
        ignore_index, reduction = ctx.args
        want_x, want_w = ctx.needs_input_grad[:2]
        dev, dim = x.device, int(x.shape[-1])
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if want_x else None
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=dev) if want_w else None
        if t.numel() == 0:
            return dx, None if dw is None else dw.zero_(), None, None, None
        xr, w = _rows(x, dim), _rows(weight, dim)
        g = grad.reshape(-1)
        if g.dtype != torch.float32:
            g = g.float()
        args = L.LinearCrossEntropyGradArgs(
            x=L.ptr(xr), weight=L.ptr(w), targets=L.ptr(t), loss=L.ptr(loss), lse=L.ptr(lse),
            grad_loss=L.ptr(g), grad_x=L.ptr(dx), grad_weight=L.ptr(dw), n=t.numel(),
            vocab=int(w.shape[0]), dim=dim, ldx=_stride(xr, dim), ldw=_stride(w, dim),
            ignore_index=ignore_index,
            grad_loss_stride=0 if reduction != "none" else int(g.stride(0)),
            dtype=L.dtype_code(w, "weight"), target_dtype=L.index_code(t, "targets"),
            mean=int(reduction == "mean"))
        L.call_with_workspace("m2_linear_cross_entropy_grad", args, dev)
        return dx, dw, None, None, None


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
    maximum and sum and the loss are float32 or wider.  The gradient computes
    the logits again, at most 512 MB of their gradient at a time: bfloat16
    operands round it to bfloat16 before its products with weight and x (float32
    sums, each result rounded once); float32 operands are multiplied as three
    bfloat16 parts each, accurate to about 2^-24 of each product."""
    dev = L.device_of(x, weight, targets)
    L.require(reduction in REDUCTIONS, f"reduction={reduction!r}: one of {REDUCTIONS}")
    L.require(weight.dim() == 2 and x.dim() >= 1 and x.shape[-1] == weight.shape[1],
              f"x.shape={tuple(x.shape)}, weight.shape={tuple(weight.shape)}: expected (..., dim) "
              "and (vocab, dim)")
    L.require(tuple(targets.shape) == tuple(x.shape[:-1]),
              f"targets.shape={tuple(targets.shape)}: expected {tuple(x.shape[:-1])}")
    L.require(weight.shape[0] > 0 and weight.shape[1] > 0, f"weight.shape={tuple(weight.shape)}")
    L.index_code(targets, "targets")
    if L.dtype_code(x, "x") != L.dtype_code(weight, "weight"):
        raise TypeError(f"x is {x.dtype} and weight {weight.dtype}: they must be the same")
    del dev
    return _LinearCrossEntropy.apply(x, weight, targets, ignore_index, reduction)


__all__ = ["linear_cross_entropy"]
