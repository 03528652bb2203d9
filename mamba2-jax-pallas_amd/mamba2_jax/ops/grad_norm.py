"""The 2-norm over many tensors and clipping by it on MI355X, as HIP kernels in
libm2ssd.so (m2_clip_grad_norm).  No counterpart in the reference, which has no
training path.
"""

from __future__ import annotations

from array import array
from itertools import chain

import torch

from .. import _lib as L


# (maps of these cost half as much per tensor as a loop that calls the methods, and a
# model has hundreds of tensors)
_ptr, _numel, _contiguous = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous
_CODES = {torch.float32: L.M2_F32, torch.bfloat16: L.M2_BF16}


def _dense(t):
    """True when t's elements fill one block of memory, in any order of dimensions."""
    return t.is_contiguous() or torch.empty_like(t, device="meta").stride() == t.stride()


def _device(tensors):
    """The common GPU device of the tensors."""
    try:
        devices = set(map(torch.Tensor.get_device, tensors))
    except TypeError:
        devices = ()
    if len(devices) == 1 and -1 not in devices:
        return tensors[0].device
    return L.device_of(*tensors)          # says what is wrong


def _gathered(tensors):
    if all(map(_contiguous, tensors)):
        return tensors
    return [t if _dense(t) else t.detach().contiguous() for t in tensors]


def _run(dev, tensors, outs, max_norm, eps):
    # a table of m2_tensor_ref (in, out, n, dtype)
    codes = [_CODES.get(t.dtype) for t in tensors]
    if None in codes:
        L.dtype_code(tensors[codes.index(None)], "a tensor")      # raises
    to = [0] * len(tensors) if outs is None else map(_ptr, outs)
    refs = array("q", chain.from_iterable(zip(map(_ptr, tensors), to, map(_numel, tensors), codes)))
    norm = torch.empty((), dtype=torch.float32, device=dev)
    args = L.ClipGradNormArgs(refs.buffer_info()[0], len(tensors), norm.data_ptr(), max_norm, eps,
                              int(outs is not None))
    L.call_with_workspace("m2_clip_grad_norm", args, dev)
    return norm


def global_norm(tensors):
    """The square root of the sum of the squares of all values of all tensors (float32
    or bfloat16, on one GPU), a float32 scalar on the GPU; summed in float64 in
    a fixed order."""
    tensors = list(tensors)
    L.require(len(tensors) > 0, "global_norm: no tensors")
    dev = _device(tensors)
    return _run(dev, _gathered(tensors), None, 0.0, 0.0)


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
    grads = list(grads)
    L.require(len(grads) > 0, "clip_grad_norm: no gradients")
    max_norm, eps = float(max_norm), float(eps)
    L.require(max_norm >= 0 and eps >= 0, lambda: f"max_norm={max_norm}, eps={eps}: must not be negative")
    if out is None:
        dev = _device(grads)
        grads = _gathered(grads)
        outs = [torch.empty_like(g, requires_grad=False) for g in grads]
    else:
        outs = list(out)
        L.require(len(outs) == len(grads),
                  lambda: f"out holds {len(outs)} tensors for {len(grads)} gradients")
        dev = _device(grads + outs)
        if not ([g.shape for g in grads] == [o.shape for o in outs]
                and [g.dtype for g in grads] == [o.dtype for o in outs]
                and all(map(_contiguous, grads)) and all(map(_contiguous, outs))):
            for i, (g, o) in enumerate(zip(grads, outs)):
                if not (o.shape == g.shape and o.dtype == g.dtype
                        and (o.is_contiguous() and g.is_contiguous()
                             or o.stride() == g.stride() and _dense(o))):
                    raise L.M2ShapeError(f"out[{i}] must have the shape, dtype and strides of its "
                                         "gradient, without gaps")
    norm = _run(dev, grads, outs, max_norm, eps)
    if out is not None:
        torch.autograd.graph.increment_version(outs)
    return outs, norm


__all__ = ["clip_grad_norm", "global_norm"]
