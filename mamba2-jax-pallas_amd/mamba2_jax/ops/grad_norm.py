"""The 2-norm over many tensors and clipping by it on MI355X, as HIP kernels in
libm2ssd.so (m2_clip_grad_norm).  No counterpart in the reference, which has no
training path.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _lib as L


def _dense(t):
    """True when t's elements fill one block of memory, in any order of dimensions."""
    return t.is_contiguous() or torch.empty_like(t, device="meta").stride() == t.stride()


def _run(tensors, outs, max_norm, eps):
    dev = L.device_of(*tensors)
    refs = (L.TensorRef * len(tensors))()
    flat = []
    for i, t in enumerate(tensors):
        flat += (t.data_ptr(), 0 if outs is None else outs[i].data_ptr(), t.numel(),
                 L.dtype_code(t, f"tensor {i}"))
    ctypes.memmove(refs, (ctypes.c_int64 * len(flat))(*flat), ctypes.sizeof(refs))
    norm = torch.empty((), dtype=torch.float32, device=dev)
    args = L.ClipGradNormArgs(tensors=ctypes.addressof(refs), count=len(tensors), norm=norm.data_ptr(),
                              max_norm=max_norm, eps=eps, clip=int(outs is not None))
    L.call_with_workspace("m2_clip_grad_norm", args, dev)
    return norm


def global_norm(tensors):
    """The square root of the sum of the squares of all values of all tensors (float32
    or bfloat16, on one GPU), a float32 scalar on the GPU; summed in float64 in
    a fixed order."""
    tensors = [t.detach() if _dense(t) else t.detach().contiguous() for t in tensors]
    L.require(len(tensors) > 0, "global_norm: no tensors")
    return _run(tensors, None, 0.0, 0.0)


def clip_grad_norm(grads, max_norm, *, out=None, eps=1e-6):
    """-> (clipped, norm): norm is the 2-norm over all values of all gradients before
    clipping (a float32 scalar on the GPU), clipped the list of grads times
    min(1, max_norm / (norm + eps)), each in its own dtype (float32 product,
    rounded once).  A norm that is not a number makes every result not a number.

    grads: float32 or bfloat16 tensors on one GPU, of any shapes.  out (keyword
    only): the tensors to write, of grads' shapes, dtypes and strides, which are
    returned; out=grads clips in place (and writes nothing where the norm is within
    max_norm).  By default the results are new tensors and grads stay as they
    are.  max_norm must not be negative."""
    grads = [g.detach() for g in grads]
    L.require(len(grads) > 0, "clip_grad_norm: no gradients")
    max_norm, eps = float(max_norm), float(eps)
    L.require(max_norm >= 0 and eps >= 0, f"max_norm={max_norm}, eps={eps}: must not be negative")
    if out is None:
        grads = [g if _dense(g) else g.contiguous() for g in grads]
        outs = [torch.empty_like(g) for g in grads]
    else:
        outs = list(out)
        L.require(len(outs) == len(grads), f"out holds {len(outs)} tensors for {len(grads)} gradients")
        for i, (g, o) in enumerate(zip(grads, outs)):
            L.require(o.shape == g.shape and o.dtype == g.dtype
                      and (o.is_contiguous() and g.is_contiguous()
                           or o.stride() == g.stride() and _dense(o)),
                      lambda: f"out[{i}] must have the shape, dtype and strides of its gradient, "
                              "without gaps")
        L.device_of(*grads, *outs)
    norm = _run(grads, outs, max_norm, eps)
    if out is not None:
        torch.autograd.graph.increment_version(outs)
    return outs, norm


__all__ = ["clip_grad_norm", "global_norm"]
