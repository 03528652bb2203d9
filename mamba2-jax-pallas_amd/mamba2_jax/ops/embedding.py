"""Embedding lookup on MI355X and its gradient by sorted tokens, as HIP kernels
in libm2ssd.so (m2_embedding, m2_embedding_grad).

No counterpart operator in the reference, whose lookup is an array index
(models/mamba2_lm.py:190): the gradient of that index under autograd is a scatter-add of
float atomics, whose order changes its result; this one sorts the tokens and
gives equal bits for equal inputs.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _lib as L


def _rows(t, dim):
    """t (..., dim) as rows (n, dim) with unit last stride (a view where it can be)."""
    if t.dim() != 2:
        t = t.reshape(-1, dim)
    if (t.shape[0] > 1 and t.stride(0) < dim) or (dim > 1 and t.stride(1) != 1):
        t = t.contiguous()
    return t


def _stride(t, dim):
    return t.stride(0) if t.shape[0] > 1 else dim


def _dense(t):
    return t if t.is_contiguous() else t.contiguous()


def _lookup(dev, ids, weight, scale):
    code, id_code = L.dtype_code(weight, "weight"), L.index_code(ids, "ids")
    vocab, dim = weight.shape
    if not (vocab and dim):
        raise L.M2ShapeError(f"weight.shape={tuple(weight.shape)}")
    ids, w = _dense(ids), _rows(weight, dim)
    out = w.new_empty((*ids.shape, dim))
    n = ids.numel()
    if n:
        args = L.EmbeddingArgs(ids.data_ptr(), w.data_ptr(), out.data_ptr(), n, vocab, dim,
                               _stride(w, dim), dim, scale, id_code, code)
        with L.on_device(dev):
            L.call("m2_embedding", args, L.stream_of(dev))
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.args = int(weight.shape[0]), scale, padding_idx, weight.dtype
        return _lookup(weight.device, ids, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        vocab, scale, padding_idx, dtype = ctx.args
        return None, embedding_grad(ids, grad, vocab, scale=scale, padding_idx=padding_idx,
                                    dtype=dtype), None, None


def _padding(padding_idx, vocab):
    if padding_idx is None:
        return None
    p = int(padding_idx)
    L.require(-vocab <= p < vocab, f"padding_idx={p} outside the vocabulary of {vocab}")
    return p % vocab


def embedding(ids, weight, scale=1.0, padding_idx=None):
    """-> scale * weight[ids], shape (*ids.shape, dim), weight's dtype (the product
    in float32, rounded once); differentiable in weight.

    ids: int32 or int64, any shape.  weight (vocab, dim) float32 or bfloat16, rows
    with a contiguous last dimension read in place.  An id outside the
    vocabulary cannot be reported without waiting for the GPU: its row is NaN,
    and it takes no part in the gradient.  padding_idx: an id whose gradient is left
    out (its row is looked up like any other)."""
    dev = L.device_of_two(weight, ids)
    if weight.dim() != 2:
        raise L.M2ShapeError(f"weight.shape={tuple(weight.shape)}: expected (vocab, dim)")
    if padding_idx is not None:
        padding_idx = _padding(padding_idx, weight.shape[0])
    scale = float(scale)
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(ids, weight, scale, padding_idx)
    L.refuse_tangents(weight)
    return _lookup(dev, ids, weight, scale)


def embedding_grad(ids, grad, num_embeddings, scale=1.0, padding_idx=None, *, dtype=None, out=None):
    """The gradient of ``embedding`` in its weight: (num_embeddings, dim), row v the
    sum of scale * grad over the positions with ids == v, in their order
    (float32 sums, rounded once; equal inputs give equal bits), zeros elsewhere.

    ids: int32 or int64; grad (*ids.shape, dim) float32 or bfloat16.  dtype
    (keyword only): float32 or bfloat16, default grad's.  out (keyword only): a
    (num_embeddings, dim) float32 or bfloat16 tensor that the rows named by
    ids are added into in place, the others left untouched, and that is returned: the
    gradient of an embedding tied to the head, after the head's."""
    dev = L.device_of_two(grad, ids) if out is None else L.device_of(ids, grad, out)
    vocab = int(num_embeddings)
    L.require(0 < vocab < 2 ** 27, lambda: f"num_embeddings={vocab}")
    L.require(grad.dim() == ids.dim() + 1 and grad.shape[:-1] == ids.shape,
              lambda: f"grad.shape={tuple(grad.shape)}: expected {tuple(ids.shape)} + (dim,)")
    dim = grad.shape[-1]
    L.require(dim > 0, "grad has no columns")
    grad_code, id_code = L.dtype_code(grad, "grad"), L.index_code(ids, "ids")
    padding_idx = _padding(padding_idx, vocab)
    ids, g = _dense(ids), _rows(grad, dim)
    accumulate = out is not None
    if accumulate:
        L.require(dtype is None or out.dtype == dtype, "dtype and out disagree")
        L.require(out.shape == (vocab, dim) and (dim == 1 or out.stride(1) == 1)
                  and (vocab == 1 or out.stride(0) >= dim),
                  f"out must be ({vocab}, {dim}) with a contiguous last dimension")
    else:
        out = g.new_empty((vocab, dim), dtype=None if dtype is None else L.torch_dtype(dtype))
    args = L.EmbeddingGradArgs(
        ids.data_ptr(), g.data_ptr(), out.data_ptr(), ids.numel(), vocab, dim, _stride(g, dim),
        _stride(out, dim), -1 if padding_idx is None else padding_idx, float(scale), id_code,
        grad_code, L.dtype_code(out, "out"), int(accumulate))
    L.call_with_workspace("m2_embedding_grad", args, dev)
    if accumulate:
        torch.autograd.graph.increment_version(out)
    return out


__all__ = ["embedding", "embedding_grad"]
