"""The gated linear recurrence over time on MI355X, its gradient and its single step, as
HIP kernels in libm2ssd.so (m2_gated_recurrence, m2_gated_recurrence_grad,
m2_gated_recurrence_update).

    log a_t = A sigmoid(r_t)
    h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(i_t) x_t

No counterpart operator in the reference, whose only recurrence is the SSD's
(ops/ssd_naive.py:220-322), a state of headdim x dstate values with one decay for each head;
here a channel is a state of its own with its own decay, and the two gates come
straight from the projections that make them.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _lib as L


def _rows(t):
    """t (batch, dim) with contiguous channels (a copy where they are not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


MAX_STRIDE = 2 ** 20


def _strided(t):
    """t (batch, seqlen, dim) as the kernels read it in place: contiguous channels, positions that are one, or
    behind each other and at most MAX_STRIDE elements apart; a copy where it is not so."""
    _, seqlen, dim = t.shape
    st = t.stride(1)
    if t.stride(2) == 1 or dim == 1:
        if st == 0 or dim <= st <= MAX_STRIDE:
            return t
        if seqlen == 1:                   # (no next position: any stride)
            return t.as_strided(t.shape, (t.stride(0), dim, 1))
    return t.contiguous()


def _f32(t):
    """t as a contiguous float32 tensor (a view where it can be), or None."""
    if t is None:
        return None
    if t.dtype != torch.float32:
        t = t.float()
    return t if t.is_contiguous() else t.contiguous()


def _forward(x, r, i, A, initial_states, seq_idx, want_final, save):
    """-> (out, the final states or None, what the gradient reads, x's, r's and i's strides in it)"""
    dev = x.device
    batch, seqlen, dim = x.shape
    x, r, i = _strided(x), _strided(r), _strided(i)
    A, h0 = _f32(A), _f32(initial_states)
    out = torch.empty((batch, seqlen, dim), dtype=x.dtype, device=dev)
    final = torch.empty((batch, dim), dtype=torch.float32, device=dev) if want_final else None
    spans = torch.empty((batch, -(-seqlen // L.RECURRENCE_SPAN), dim), dtype=torch.float32, device=dev) \
        if save else None
    strides = sx, sr, si = x.stride(), r.stride(), i.stride()
    args = L.GatedRecurrenceArgs(
        x.data_ptr(), r.data_ptr(), i.data_ptr(), A.data_ptr(), L.ptr(h0), L.ptr(seq_idx),
        out.data_ptr(), L.ptr(final), L.ptr(spans), batch, seqlen, dim, sx[0], sx[1], sr[0], sr[1], si[0], si[1],
        L.dtype_code(x, "x"))
    L.call_with_workspace("m2_gated_recurrence", args, dev)
    return out, final, (x, r, i, A, seq_idx, spans), strides


def _saved(ctx):
    """What the forward saved, as the kernels read it: hooks may have given it back at other places and strides."""
    x, r, i, A, seq_idx, spans = saved = ctx.saved_tensors
    shape, dtype, spans_shape, strides = ctx.saved_as
    _device(*saved)
    if not (x.shape == r.shape == i.shape == shape and x.dtype == r.dtype == i.dtype == dtype and A.dtype == torch.float32
            and A.shape == shape[2:] and spans.shape == spans_shape and spans.dtype == torch.float32
            and (seq_idx is None or (seq_idx.shape == shape[:2] and seq_idx.dtype == torch.int32))):
        for t in (x, r, i):
            L.require_saved(t, shape, dtype, "x, r or i")
        L.require_saved(A, shape[2:], torch.float32, "A")
        L.require_saved(spans, spans_shape, torch.float32, "span states")
        L.require_saved(seq_idx, shape[:2], torch.int32, "seq_idx")
    if seq_idx is not None:
        seq_idx = seq_idx.contiguous()
    if (x.stride(), r.stride(), i.stride()) != strides:
        x, r, i = _strided(x), _strided(r), _strided(i)
        strides = x.stride(), r.stride(), i.stride()
    return x, r, i, A.contiguous(), seq_idx, spans.contiguous(), strides


def _backward(ctx, grad, grad_final=None):
    x, r, i, A, seq_idx, spans, (sx, sr, si) = _saved(ctx)
    a_dtype, h0_dtype = ctx.dtypes
    batch, seqlen, dim = x.shape
    dev = x.device
    has_h0 = h0_dtype is not None
    if batch == 0 or seqlen == 0:
        dh0 = None
        if has_h0:
            dh0 = torch.zeros((batch, dim), dtype=h0_dtype, device=dev) if grad_final is None \
                else grad_final.to(h0_dtype)
        return x.new_zeros(x.shape), x.new_zeros(x.shape), x.new_zeros(x.shape), \
            torch.zeros(dim, dtype=a_dtype, device=dev), dh0, None, None
    g = x.new_zeros(x.shape) if grad is None else _strided(grad)
    gf = _f32(grad_final)
    dx, dr, di = (torch.empty((batch, seqlen, dim), dtype=x.dtype, device=dev) for _ in range(3))
    dA = torch.empty(dim, dtype=torch.float32, device=dev)
    dh0 = torch.empty((batch, dim), dtype=torch.float32, device=dev) if has_h0 else None
    args = L.GatedRecurrenceGradArgs(
        x.data_ptr(), r.data_ptr(), i.data_ptr(), A.data_ptr(), L.ptr(seq_idx), spans.data_ptr(),
        g.data_ptr(), L.ptr(gf), dx.data_ptr(), dr.data_ptr(), di.data_ptr(), dA.data_ptr(),
        L.ptr(dh0), batch, seqlen, dim, sx[0], sx[1], sr[0], sr[1], si[0], si[1], g.stride(0), g.stride(1),
        L.dtype_code(x, "x"))
    L.call_with_workspace("m2_gated_recurrence_grad", args, dev)
    if a_dtype != torch.float32:
        dA = dA.to(a_dtype)
    if has_h0 and h0_dtype != torch.float32:
        dh0 = dh0.to(h0_dtype)
    return dx, dr, di, dA, dh0, None, None


_backward_once = once_differentiable(_backward)


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, r, i, A, initial_states, seq_idx, want_final):
        ctx.set_materialize_grads(False)
        out, final, saved, strides = _forward(x, r, i, A, initial_states, seq_idx, want_final, True)
        ctx.save_for_backward(*saved)
        ctx.saved_as = x.shape, x.dtype, saved[5].shape, strides
        ctx.dtypes = A.dtype, None if initial_states is None else initial_states.dtype
        return (out, final) if want_final else out

    @staticmethod
    def backward(ctx, grad, grad_final=None):
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, grad, grad_final)


def _device(*tensors):
    """L.device_of(*tensors), without its cost where all is well."""
    try:
        at = tensors[0].get_device()
        if at >= 0:
            for t in tensors:
                if t is not None and t.get_device() != at:
                    break
            else:
                return tensors[0].device
    except AttributeError:
        pass
    return L.device_of(*tensors)          # says what is wrong


def _check_gates(x, r, i, A, shape):
    """-> x's type code"""
    if not (r.shape == shape and i.shape == shape and shape[-1] > 0 and A.shape == shape[-1:]):
        L.require(shape[-1] > 0, f"x.shape={tuple(shape)}: no channels")
        raise L.M2ShapeError(f"r.shape={tuple(r.shape)}, i.shape={tuple(i.shape)}, A.shape={tuple(A.shape)}: "
                             f"expected x's {tuple(shape)} and ({shape[-1]},)")
    dtype = x.dtype
    code = L.dtype_code(x, "x")
    if r.dtype != dtype or i.dtype != dtype:
        raise TypeError(f"x is {dtype}, r {r.dtype} and i {i.dtype}: they must be the same")
    L.dtype_code(A, "A")
    return code


def gated_linear_recurrence(x, r, i, A, initial_states=None, seq_idx=None, return_final_states=False):
    """-> h (batch, seqlen, dim), x's dtype, and with return_final_states (h, final states (batch,
    dim) float32), of

        log a_t = A sigmoid(r_t),  h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(i_t) x_t

    for every channel; differentiable in x, r, i, A and initial_states.

    x, r, i (batch, seqlen, dim), all bfloat16 or all float32: views whose channels are
    contiguous (slices of one projection's output, say) are read in place.  A (dim,), finite and <= 0 (a
    positive one gives NaN), float32 or bfloat16.  initial_states (batch, dim): h_{-1}, zeros by
    default.  seq_idx (batch, seqlen) int32 or int64 (of int32's range): where an entry differs from the one before it a new
    sequence begins, with a state of zero (the one at a row's first position goes on from initial_states); a negative
    entry is padding: h is 0 there, the state passes it unchanged, its
    gradients are 0 and what the inputs hold there (a NaN, say) reaches nothing.  An entry behind padding differs from
    it and begins a sequence: a row that begins with padding has no use for initial_states but as final states of
    padding alone.  The final
    states are those behind the last position.

    Gates, states and sums are float32 (a state and the gradient that comes back to it never
    leave it between two positions); h and the gradients are rounded once.  Between the two the graph holds x, r, i and
    the states that enter every 32 positions.  Where a_t is 1 the root has no slope, and its part
    of the gradient is taken as 0.  a_t is never 0: an infinite state (or gradient of one) stays infinite until its sequence
    ends.  Inputs that carry forward-mode derivatives are refused.  Equal inputs give equal bits."""
    dev = _device(x, r, i, A, initial_states, seq_idx)
    shape = x.shape
    L.require(len(shape) == 3, lambda: f"x.shape={tuple(shape)}: expected (batch, seqlen, dim)")
    _check_gates(x, r, i, A, shape)
    L.require(shape[2] <= MAX_STRIDE, lambda: f"x.shape={tuple(shape)}: more than {MAX_STRIDE} channels")
    if initial_states is not None:
        L.require(initial_states.shape == (shape[0], shape[2]),
                  lambda: f"initial_states.shape={tuple(initial_states.shape)}: expected {(shape[0], shape[2])}")
        L.dtype_code(initial_states, "initial_states")
    if seq_idx is not None:
        L.require(seq_idx.shape == shape[:2],
                  lambda: f"seq_idx.shape={tuple(seq_idx.shape)}: expected {tuple(shape[:2])}")
        L.index_code(seq_idx, "seq_idx")
        seq_idx = seq_idx.to(torch.int32).contiguous()
    want_final = bool(return_final_states)
    if torch.is_grad_enabled() and (x.requires_grad or r.requires_grad or i.requires_grad or A.requires_grad
                                    or (initial_states is not None and initial_states.requires_grad)):
        return _GatedRecurrence.apply(x, r, i, A, initial_states, seq_idx, want_final)
    L.refuse_tangents(x, r, i, A, initial_states)
    out, final, _, _ = _forward(x, r, i, A, initial_states, seq_idx, want_final, False)
    return (out, final) if want_final else out


def gated_linear_recurrence_update(state, x, r, i, A, *, inplace=False):
    """One step of ``gated_linear_recurrence`` -> (new_state (batch, dim) float32, h (batch, dim),
    x's dtype).

    state (batch, dim), batch at most 65535; x, r, i (batch, dim), all bfloat16 or all float32, rows with contiguous
    channels read in place; A (dim,).  The caller's state is left untouched, unless inplace=True (keyword
    only) and it is float32 and contiguous: it is then updated and returned.
    Takes no gradients: an input that requires one is refused where they are recorded."""
    dev = _device(state, x, r, i, A)
    shape = x.shape
    if len(shape) != 2 or state.shape != shape:
        raise L.M2ShapeError(f"x.shape={tuple(shape)}, state.shape={tuple(state.shape)}: expected (batch, dim)")
    code = _check_gates(x, r, i, A, shape)
    L.dtype_code(state, "state")
    L.refuse_tangents(state, x, r, i, A)
    if torch.is_grad_enabled() and (state.requires_grad or x.requires_grad or r.requires_grad or i.requires_grad
                                    or A.requires_grad):
        raise L.M2ShapeError("a single step takes no gradients: call it under torch.no_grad(), or gated_linear_recurrence")
    src = _f32(state)
    new = src if inplace and src is state else torch.empty(shape, dtype=torch.float32, device=dev)
    if not (x.stride(1) == r.stride(1) == i.stride(1) == 1):
        x, r, i = _rows(x), _rows(r), _rows(i)
    A = _f32(A)
    out = torch.empty(shape, dtype=x.dtype, device=dev)
    args = L.GatedRecurrenceUpdateArgs(
        x.data_ptr(), r.data_ptr(), i.data_ptr(), A.data_ptr(), src.data_ptr(), new.data_ptr(),
        out.data_ptr(), shape[0], shape[1], x.stride(0), r.stride(0), i.stride(0), code)
    with L.on_device(dev):
        L.call("m2_gated_recurrence_update", args, L.stream_of(dev))
    if new is state:
        torch.autograd.graph.increment_version(new)
    return new, out


__all__ = ["gated_linear_recurrence", "gated_linear_recurrence_update"]
