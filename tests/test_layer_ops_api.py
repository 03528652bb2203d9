"""Refusals of the operators of a trained layer, and the layout of their argument structs, without a GPU."""

import ctypes
import os
import re
import subprocess

import pytest
import torch

from mamba2_jax import _lib as L
from mamba2_jax import ops

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "m2ssd.h")
STRUCTS = {"GatedRecurrenceArgs": "m2_gated_recurrence_args",
           "GatedRecurrenceGradArgs": "m2_gated_recurrence_grad_args",
           "GatedRecurrenceUpdateArgs": "m2_gated_recurrence_update_args",
           "GatedLinearArgs": "m2_gated_linear_args", "GatedLinearGradArgs": "m2_gated_linear_grad_args"}


def test_struct_layout_matches_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void) {"]
    for py, c in STRUCTS.items():
        lines.append(f'printf("{py} %zu\\n", sizeof({c}));')
        for f, _ in getattr(L, py)._fields_:
            lines.append(f'printf("{py}.{f} %zu\\n", offsetof({c}, {f}));')
    lines.append('printf("span %d\\n", M2_RECURRENCE_SPAN);')
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", str(src), "-o", str(tmp_path / "probe")], check=True)
    got = dict(l.rsplit(" ", 1) for l in subprocess.run(
        [str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(got["span"]) == L.RECURRENCE_SPAN
    for py in STRUCTS:
        st = getattr(L, py)
        assert int(got[py]) == ctypes.sizeof(st), py
        for f, _ in st._fields_:
            assert int(got[f"{py}.{f}"]) == getattr(st, f).offset, f"{py}.{f}"


def refused(name, args, code, text):
    lib = L.load_library()
    assert getattr(lib, name)(ctypes.byref(args), None) == code
    assert text in lib.m2_last_error().decode()


def test_gated_recurrence_refusals():
    ok = dict(x=4096, r=4096, i=4096, A=4096, out=4096, batch=2, seqlen=9, dim=8, x_stride_batch=72, x_stride_time=8,
              r_stride_batch=72, r_stride_time=8, i_stride_batch=72, i_stride_time=8, dtype=L.M2_BF16)
    mk = lambda **k: L.GatedRecurrenceArgs(**{**ok, **k})
    name = "m2_gated_recurrence"
    for bad in (dict(batch=-1), dict(seqlen=-1), dict(dim=0), dict(dim=(1 << 20) + 1), dict(seqlen=1 << 40)):
        refused(name, mk(**bad), -1, "bad sizes")
    refused(name, mk(dtype=L.M2_I32), -2, "dtype")
    refused(name, mk(batch=1 << 31, dim=64), -2, "too many rows")
    refused(name, mk(batch=1 << 22, dim=1), -2, "too many rows")
    refused(name, mk(batch=1 << 12, dim=1 << 16), -2, "too many rows")
    refused(name, mk(batch=1 << 21, seqlen=1 << 12, dim=1), -2, "too many steps")
    refused(name, mk(seqlen=65536), -4, "workspace")
    refused(name, mk(seqlen=65536, workspace=4104, workspace_bytes=1 << 30), -4, "alignment")
    assert L.load_library().m2_gated_recurrence_workspace_size(ctypes.byref(mk(seqlen=65536))) > 0
    for p in ("x", "r", "i", "A", "out"):
        refused(name, mk(**{p: None}), -1, "required")
    for p in "xri":
        for st in (-8, 7, (1 << 20) + 1):
            refused(name, mk(**{p + "_stride_time": st}), -1, "strides of time")
    okg = {k: v for k, v in ok.items() if k != "out"} | dict(
        span_states=4096, grad_out=4096, grad_x=4096, grad_r=4096, grad_i=4096, grad_A=4096,
        grad_out_stride_batch=72, grad_out_stride_time=8)
    mg = lambda **k: L.GatedRecurrenceGradArgs(**{**okg, **k})
    lib = L.load_library()
    need = lib.m2_gated_recurrence_grad_workspace_size(ctypes.byref(mg()))
    assert need > 0
    assert lib.m2_gated_recurrence_grad_workspace_size(ctypes.byref(mg(dim=0))) == 0
    name = "m2_gated_recurrence_grad"
    refused(name, mg(batch=0), -1, "no steps")
    refused(name, mg(seqlen=0), -1, "no steps")
    refused(name, mg(dtype=7), -2, "dtype")
    for p in ("x", "r", "i", "A", "span_states", "grad_out", "grad_x", "grad_r", "grad_i", "grad_A"):
        refused(name, mg(**{p: None}), -1, "required")
    refused(name, mg(grad_out_stride_time=7), -1, "strides of time")
    refused(name, mg(workspace=4096, workspace_bytes=need - 1), -4, "workspace")
    refused(name, mg(workspace=4104, workspace_bytes=need), -4, "alignment")
    refused(name, mg(workspace_bytes=need), -4, "workspace")


def test_gated_recurrence_update_refusals():
    ok = dict(x=4096, r=4096, i=4096, A=4096, state=4096, new_state=4096, out=4096, batch=2, dim=8, x_stride_batch=8,
              r_stride_batch=8, i_stride_batch=8, dtype=L.M2_F32)
    mk = lambda **k: L.GatedRecurrenceUpdateArgs(**{**ok, **k})
    name = "m2_gated_recurrence_update"
    refused(name, mk(dim=0), -1, "bad sizes")
    refused(name, mk(dtype=3), -2, "dtype")
    refused(name, mk(batch=65536), -2, "batch")
    for p in ("x", "r", "i", "A", "state", "new_state", "out"):
        refused(name, mk(**{p: None}), -1, "required")
    assert L.load_library().m2_gated_recurrence_update(ctypes.byref(mk(batch=0, x=None)), None) == 0


def test_gated_linear_refusals():
    ok = dict(x=4096, weight=4096, out=4096, n=100, dim=60, hidden=30, ldx=60, ldw=60, dtype=L.M2_BF16,
              activation=L.ACTIVATIONS["silu"])
    mk = lambda **k: L.GatedLinearArgs(**{**ok, **k})
    lib = L.load_library()
    name = "m2_gated_linear"
    need = lib.m2_gated_linear_workspace_size(ctypes.byref(mk()))
    saved = lib.m2_gated_linear_saved_size(ctypes.byref(mk()))
    assert need > 0 and saved >= 100 * 2 * 64 * 2
    far = dict(ldx=1 << 22, ldw=1 << 22)
    for bad in (dict(n=-1), dict(n=1 << 30), dict(dim=0), dict(dim=1 << 21), dict(hidden=0), dict(hidden=1 << 28)):
        assert lib.m2_gated_linear_workspace_size(ctypes.byref(mk(**{**far, **bad}))) == 0
        assert lib.m2_gated_linear_saved_size(ctypes.byref(mk(**{**far, **bad}))) == 0
        refused(name, mk(**{**far, **bad}), -1, "bad sizes")
    refused(name, mk(ldx=59), -1, "row strides")
    refused(name, mk(ldw=59), -1, "row strides")
    refused(name, mk(dtype=L.M2_I64), -2, "dtype")
    refused(name, mk(activation=2), -2, "activation")
    refused(name, mk(dim=1 << 16, ldx=1 << 16, ldw=1 << 16, hidden=1 << 14), -2, "too large")
    refused(name, mk(hidden=(1 << 21) + 1), -2, "too large")
    for p in ("x", "weight", "out"):
        refused(name, mk(**{p: None}), -1, "required")
    refused(name, mk(workspace=4096, workspace_bytes=need - 1), -4, "workspace")
    refused(name, mk(workspace_bytes=need), -4, "workspace")
    refused(name, mk(workspace=4096, workspace_bytes=need, saved=4096, saved_bytes=saved - 1), -4, "saved")
    refused(name, mk(workspace=4096, workspace_bytes=need, saved=4104, saved_bytes=saved), -4, "alignment")
    refused(name, mk(workspace=4104, workspace_bytes=need), -4, "alignment")
    assert lib.m2_gated_linear(ctypes.byref(mk(n=0, x=None)), None) == 0
    okg = {k: v for k, v in ok.items() if k != "out"} | dict(saved=4096, saved_bytes=saved, grad_out=4096, grad_x=4096,
                                                            grad_weight=4096, ldg=30)
    mg = lambda **k: L.GatedLinearGradArgs(**{**okg, **k})
    name = "m2_gated_linear_grad"
    need = lib.m2_gated_linear_grad_workspace_size(ctypes.byref(mg()))
    assert need > 0
    refused(name, mg(n=0), -1, "no tokens")
    refused(name, mg(ldg=29), -1, "row strides")
    for p in ("x", "weight", "saved", "grad_out"):
        refused(name, mg(**{p: None}), -1, "required")
    refused(name, mg(grad_x=None, grad_weight=None), -1, "required")
    refused(name, mg(workspace=4096, workspace_bytes=need, saved_bytes=saved - 1), -4, "saved")
    refused(name, mg(workspace=4096, workspace_bytes=need - 1), -4, "workspace")


def test_gated_linear_saved_layouts():
    """What lies in `saved` follows from its size alone, wherever x and weight lie when the gradient is taken; a size that is no
    forward's is refused."""
    lib = L.load_library()
    n, dim, hidden = 512, 256, 256              # (as many rows of x as weight has)
    sizes = set()
    for x in (4096, 4098):
        for w in (4096, 4098):
            a = L.GatedLinearArgs(x=x, weight=w, out=4096, n=n, dim=dim, hidden=hidden, ldx=dim, ldw=dim, dtype=L.M2_BF16)
            sizes.add(lib.m2_gated_linear_saved_size(ctypes.byref(a)))
    assert len(sizes) == 4
    grad = lambda **k: L.GatedLinearGradArgs(**{**dict(
        x=4096, weight=4096, saved=4096, grad_out=4096, grad_x=4096, grad_weight=4096, n=n, dim=dim, hidden=hidden, ldx=dim, ldw=dim,
        ldg=hidden, dtype=L.M2_BF16), **k})
    bare = min(sizes)
    for size in sizes:
        for x, w in ((4096, 4096), (4098, 4098)):
            args = grad(x=x, weight=w, saved_bytes=size)
            assert lib.m2_gated_linear_grad_workspace_size(ctypes.byref(args)) > 0
            refused("m2_gated_linear_grad", args, -4, "workspace of")
            args.saved_bytes += 1
            refused("m2_gated_linear_grad", args, -4, "saved of")
    # what is neither there nor readable in place is packed
    ws = lambda **k: lib.m2_gated_linear_grad_workspace_size(ctypes.byref(grad(**k)))
    assert ws(saved_bytes=bare, x=4098, weight=4098) >= ws(saved_bytes=bare) + 2 * 2 * n * dim
    assert ws(saved_bytes=max(sizes), x=4098, weight=4098) == ws(saved_bytes=max(sizes)) == ws(saved_bytes=bare)


def test_gated_linear_shape_refusals():
    x, w = _fake(3, 8), _fake(12, 8)
    for args in ((x[0, 0], w), (x, w[0]), (x, w[:, :7]), (x, w[:11]), (x, w[:0]), (x[:, :0], w[:, :0]), (x, w, "relu")):
        with pytest.raises(L.M2ShapeError):
            ops.gated_linear(*args)
    with pytest.raises(TypeError):
        ops.gated_linear(x.bfloat16(), w)
    with pytest.raises(TypeError):
        ops.gated_linear(x.half(), w.half())
    with pytest.raises(ValueError):
        ops.gated_linear(torch.zeros(3, 8), torch.zeros(12, 8))


def test_python_refuses_cpu_tensors():
    x, A = torch.zeros((1, 4, 8)), torch.zeros(8)
    with pytest.raises(ValueError):
        ops.gated_linear_recurrence(x, x, x, A)
    with pytest.raises(ValueError):
        ops.gated_linear_recurrence_update(x[:, 0], x[:, 0], x[:, 0], x[:, 0], A)


class _Fake(torch.Tensor):
    """A CPU tensor that says it is on a GPU: the checks of shapes and types come before any GPU work."""

    @property
    def is_cuda(self):
        return True


def _fake(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(_Fake)


def test_python_shape_refusals():
    x, A = _fake(2, 4, 8), _fake(8)
    bad = L.M2ShapeError
    rec = ops.gated_linear_recurrence
    for args in ((x[0], x[0], x[0], A), (x, x[:, :3], x, A), (x, x, x[..., :7], A), (x, x, x, A[:7]),
                 (x, x, x, A, x[:, 0, :7]), (x, x, x, A, x[:1, 0])):
        with pytest.raises(bad):
            rec(*args)
    with pytest.raises(bad):
        rec(x, x, x, A, None, _fake(2, 3, dtype=torch.int32))
    with pytest.raises(TypeError):
        rec(x, x, x, A, None, _fake(2, 4))
    with pytest.raises(TypeError):
        rec(x, x.bfloat16(), x, A)
    with pytest.raises(TypeError):
        rec(x.half(), x.half(), x.half(), A)
    with pytest.raises(TypeError):
        rec(x, x, x, A.double())
    with pytest.raises(TypeError):
        rec(x, x, x, A, x[:, 0].half())
    with pytest.raises(bad):
        rec(x[..., :0], x[..., :0], x[..., :0], A[:0])
    step = ops.gated_linear_recurrence_update
    s = x[:, 0]
    for args in ((s, x, x, x, A), (s[:1], s, s, s, A), (s, s, s[:1], s, A), (s, s, s, s, A[:3])):
        with pytest.raises(bad):
            step(*args)
    with pytest.raises(TypeError):
        step(s.half(), s, s, s, A)
