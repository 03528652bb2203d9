"""Refusals of the vocabulary's operators, and the layout of their argument structs,
without a GPU."""

import ctypes
import os
import subprocess

import pytest
import torch

from mamba2_jax import _lib as L
from mamba2_jax import ops

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "m2ssd.h")
STRUCTS = {"EmbeddingArgs": "m2_embedding_args", "EmbeddingGradArgs": "m2_embedding_grad_args",
           "LinearCrossEntropyArgs": "m2_linear_cross_entropy_args",
           "LinearCrossEntropyGradArgs": "m2_linear_cross_entropy_grad_args",
           "TensorRef": "m2_tensor_ref", "ClipGradNormArgs": "m2_clip_grad_norm_args"}


def test_struct_layout_matches_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void) {"]
    for py, c in STRUCTS.items():
        lines.append(f'printf("{py} %zu\\n", sizeof({c}));')
        for f, _ in getattr(L, py)._fields_:
            lines.append(f'printf("{py}.{f} %zu\\n", offsetof({c}, {f.rstrip("_")}));')
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", str(src), "-o", str(tmp_path / "probe")], check=True)
    got = dict(l.rsplit(" ", 1) for l in subprocess.run(
        [str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout.splitlines())
    for py in STRUCTS:
        st = getattr(L, py)
        assert int(got[py]) == ctypes.sizeof(st), py
        for f, _ in st._fields_:
            assert int(got[f"{py}.{f}"]) == getattr(st, f).offset, f"{py}.{f}"


def refused(name, args, code, text):
    lib = L.load_library()
    assert getattr(lib, name)(ctypes.byref(args), None) == code
    assert text in lib.m2_last_error().decode()


def test_embedding_refusals():
    ok = dict(ids=4096, weight=4096, out=4096, n=4, vocab=10, dim=8, ldw=8, ldo=8, scale=1.0,
              id_dtype=L.M2_I64, dtype=L.M2_BF16)
    mk = lambda **k: L.EmbeddingArgs(**{**ok, **k})
    refused("m2_embedding", mk(vocab=0), -1, "bad sizes")
    refused("m2_embedding", mk(n=-1), -1, "bad sizes")
    refused("m2_embedding", mk(ldw=7), -1, "row strides")
    refused("m2_embedding", mk(dtype=L.M2_I32), -2, "dtype")
    refused("m2_embedding", mk(id_dtype=L.M2_F32), -2, "id dtype")
    refused("m2_embedding", mk(out=None), -1, "required")
    assert L.load_library().m2_embedding(ctypes.byref(mk(n=0, ids=None, out=None)), None) == 0


def test_embedding_grad_refusals():
    ok = dict(ids=4096, grad=4096, out=4096, n=4, vocab=10, dim=8, ldg=8, ldo=8, padding_idx=-1, scale=1.0,
              id_dtype=L.M2_I64, grad_dtype=L.M2_BF16, out_dtype=L.M2_F32)
    mk = lambda **k: L.EmbeddingGradArgs(**{**ok, **k})
    lib = L.load_library()
    need = lib.m2_embedding_grad_workspace_size(ctypes.byref(mk()))
    assert need > 0
    for bad in (dict(vocab=0), dict(vocab=2 ** 27), dict(n=-1), dict(n=2 ** 31), dict(dim=0)):
        assert lib.m2_embedding_grad_workspace_size(ctypes.byref(mk(**bad))) == 0
        refused("m2_embedding_grad", mk(**bad, workspace=4096, workspace_bytes=1 << 40), -1, "bad sizes")
    refused("m2_embedding_grad", mk(workspace=4096, workspace_bytes=need - 1), -4, "workspace")
    refused("m2_embedding_grad", mk(workspace_bytes=need), -4, "workspace")
    refused("m2_embedding_grad", mk(out_dtype=L.M2_I64), -2, "dtype")
    refused("m2_embedding_grad", mk(ldg=4), -1, "row strides")
    refused("m2_embedding_grad", mk(grad=None), -1, "required")


def test_linear_cross_entropy_refusals():
    ok = dict(x=4096, weight=4096, targets=4096, loss=4096, lse=4096, n=4, vocab=10, dim=8, ldx=8, ldw=8,
              dtype=L.M2_BF16, target_dtype=L.M2_I64)
    mk = lambda **k: L.LinearCrossEntropyArgs(**{**ok, **k})
    lib = L.load_library()
    need = lib.m2_linear_cross_entropy_workspace_size(ctypes.byref(mk()))
    assert need > 0
    for bad in (dict(vocab=0), dict(n=-1), dict(dim=0), dict(n=1 << 30), dict(vocab=1 << 30), dict(dim=1 << 21)):
        assert lib.m2_linear_cross_entropy_workspace_size(ctypes.byref(mk(**{**bad, "ldx": 1 << 22, "ldw": 1 << 22}))) == 0
        refused("m2_linear_cross_entropy", mk(**{**bad, "ldx": 1 << 22, "ldw": 1 << 22}), -1, "bad sizes")
    refused("m2_linear_cross_entropy", mk(ldx=7), -1, "row strides")
    refused("m2_linear_cross_entropy", mk(dtype=3), -2, "dtype")
    refused("m2_linear_cross_entropy", mk(target_dtype=0), -2, "target dtype")
    refused("m2_linear_cross_entropy", mk(targets=None), -1, "required")
    refused("m2_linear_cross_entropy", mk(workspace=4096, workspace_bytes=need - 1), -4, "workspace")
    okg = {k: v for k, v in ok.items()} | dict(grad_loss=4096, grad_x=4096, grad_weight=4096)
    mg = lambda **k: L.LinearCrossEntropyGradArgs(**{**okg, **k})
    need = lib.m2_linear_cross_entropy_grad_workspace_size(ctypes.byref(mg()))
    assert need > 0
    refused("m2_linear_cross_entropy_grad", mg(n=0), -1, "no tokens")
    refused("m2_linear_cross_entropy_grad", mg(grad_x=None, grad_weight=None), -1, "an output")
    refused("m2_linear_cross_entropy_grad", mg(grad_loss_stride=-1), -1, "stride")
    refused("m2_linear_cross_entropy_grad", mg(workspace=4096, workspace_bytes=need - 1), -4, "workspace")


def test_clip_refusals():
    lib = L.load_library()
    ref = (L.TensorRef * 1)(L.TensorRef(in_=4096, out=4096, n=10, dtype=L.M2_F32))
    ok = dict(tensors=ctypes.addressof(ref), count=1, norm=4096, max_norm=1.0, eps=1e-6, clip=1, workspace=4096,
              workspace_bytes=1 << 30)
    mk = lambda **k: L.ClipGradNormArgs(**{**ok, **k})
    need = lib.m2_clip_grad_norm_workspace_size(ctypes.byref(mk()))
    assert need > 0 and lib.m2_clip_grad_norm_workspace_size(ctypes.byref(mk(count=-1))) == 0
    refused("m2_clip_grad_norm", mk(count=-1), -1, "required")
    refused("m2_clip_grad_norm", mk(norm=None), -1, "required")
    refused("m2_clip_grad_norm", mk(workspace_bytes=need - 1), -4, "workspace")
    refused("m2_clip_grad_norm", mk(max_norm=-1.0), -1, "max_norm")
    refused("m2_clip_grad_norm", mk(max_norm=float("nan")), -1, "max_norm")
    ref[0].dtype = L.M2_I32
    refused("m2_clip_grad_norm", mk(), -2, "dtype")
    ref[0].dtype, ref[0].out = L.M2_F32, 4098
    refused("m2_clip_grad_norm", mk(), -1, "bad pointer")
    ref[0].out, ref[0].n = 4096, -1
    refused("m2_clip_grad_norm", mk(), -1, "bad pointer")


def test_python_refuses_cpu_tensors():
    x, w, t = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.long)
    for call in (lambda: ops.linear_cross_entropy(x, w, t), lambda: ops.embedding(t, w),
                 lambda: ops.embedding_grad(t, x, 5), lambda: ops.clip_grad_norm([x], 1.0),
                 lambda: ops.global_norm([x])):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    for call in (lambda: ops.clip_grad_norm([], 1.0), lambda: ops.global_norm([]),
                 lambda: ops.clip_grad_norm([x], -1.0), lambda: ops.clip_grad_norm([x], 1.0, out=[])):
        with pytest.raises(L.M2ShapeError):
            call()


@pytest.mark.gpu
def test_python_refuses_bad_arguments():
    x, w = torch.zeros(3, 8, device="cuda"), torch.zeros(5, 8, device="cuda")
    t = torch.zeros(3, dtype=torch.long, device="cuda")
    shape = [lambda: ops.linear_cross_entropy(x, w[:, :4], t), lambda: ops.linear_cross_entropy(x, w, t[:2]),
             lambda: ops.linear_cross_entropy(x, w, t, reduction="max"),
             lambda: ops.linear_cross_entropy(x, w[:0], t), lambda: ops.embedding(t, x[0]),
             lambda: ops.embedding(t, w, padding_idx=5), lambda: ops.embedding_grad(t, x[:2], 5),
             lambda: ops.embedding_grad(t, x, 0), lambda: ops.embedding_grad(t, x, 5, out=w[:4]),
             lambda: ops.embedding_grad(t, x, 5, out=torch.zeros(8, 5, device="cuda").t()),
             lambda: ops.clip_grad_norm([x], 1.0, out=[w]),
             lambda: ops.clip_grad_norm([x[:, ::2]], 1.0, out=[x[:, ::2]])]
    for call in shape:
        with pytest.raises(L.M2ShapeError):
            call()
    types = [lambda: ops.linear_cross_entropy(x.half(), w.half(), t),
             lambda: ops.linear_cross_entropy(x, w.bfloat16(), t), lambda: ops.linear_cross_entropy(x, w, t.float()),
             lambda: ops.embedding(t.float(), w), lambda: ops.embedding(t, w.double()),
             lambda: ops.embedding_grad(t, x.half(), 5), lambda: ops.clip_grad_norm([x.half()], 1.0)]
    for call in types:
        with pytest.raises(TypeError):
            call()
