"""What the operators of a trained layer, and the vocabulary's, refuse rather than answer without a derivative or past their
launches' counts, without a GPU."""

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from mamba2_jax import _lib as L
from mamba2_jax import ops
from test_layer_ops_api import _fake, refused


def test_forward_mode_derivatives_are_refused():
    """An output without a tangent would read as a derivative of zero."""
    x3, x2, A, w = _fake(2, 4, 8), _fake(3, 8), _fake(8), _fake(12, 8)
    ids = torch.zeros(3, dtype=torch.int64).as_subclass(type(x3))
    calls = [
        (ops.gated_linear_recurrence, (x3, x3, x3, A, x3[:, 0].clone()), range(5)),
        (ops.gated_linear_recurrence_update, (x2, x2, x2, x2, A), range(5)),
        (ops.gated_linear, (x2, w), range(2)),
        (ops.linear_cross_entropy, (x2, w, ids), range(2)),
        (ops.embedding, (ids, w), [1]),
    ]
    with fwAD.dual_level():
        for fn, args, at in calls:
            for k in at:
                dual = fwAD.make_dual(args[k].clone(), torch.ones_like(args[k]))
                with pytest.raises(NotImplementedError, match="forward"):
                    fn(*args[:k], dual, *args[k + 1:])


def test_update_refuses_inputs_that_require_gradients():
    """It takes no gradients: results without a graph would train nothing, and say nothing."""
    x, A = _fake(3, 8), _fake(8)
    for k in range(5):
        args = [x.clone() for _ in range(4)] + [A.clone()]
        args[k].requires_grad_()
        with pytest.raises(L.M2ShapeError, match="no gradients"):
            ops.gated_linear_recurrence_update(*args)


def test_cross_entropy_refuses_more_rows_than_a_launch_counts():
    """Packing takes a wavefront a row: 2^32 threads are not launched, and no kernel reads what none filled."""
    ok = dict(x=4096, weight=4096, targets=4096, loss=4096, n=100, vocab=70, dim=60, ldx=60, ldw=60, dtype=L.M2_BF16,
              target_dtype=L.M2_I32)
    mk = lambda **k: L.LinearCrossEntropyArgs(**{**ok, **k})
    lib = L.load_library()
    for bad in (dict(n=1 << 26), dict(vocab=1 << 26), dict(n=1 << 29)):
        refused("m2_linear_cross_entropy", mk(**bad), -2, "too many rows")
        assert lib.m2_linear_cross_entropy_workspace_size(ctypes.byref(mk(**bad))) == 0
    assert lib.m2_linear_cross_entropy_workspace_size(ctypes.byref(mk(n=(1 << 26) - 4096))) > 0


def test_gated_linear_grad_refuses_more_rows_than_a_launch_counts():
    lib = L.load_library()
    for n, code, text in (((1 << 28) - 300, -4, "workspace of"), (1 << 28, -2, "too many tokens"), (1 << 29, -2, "too many tokens")):
        a = L.GatedLinearArgs(x=4096, weight=4096, out=4096, n=n, dim=1, hidden=1, ldx=1, ldw=1, dtype=L.M2_BF16)
        saved = lib.m2_gated_linear_saved_size(ctypes.byref(a))
        refused("m2_gated_linear_grad", L.GatedLinearGradArgs(
            x=4096, weight=4096, saved=4096, saved_bytes=saved, grad_out=4096, grad_x=4096, grad_weight=4096, n=n, dim=1, hidden=1,
            ldx=1, ldw=1, ldg=1, dtype=L.M2_BF16), code, text)


@pytest.fixture
def recorded(monkeypatch):
    """The arguments of every launch, none of which takes place."""
    calls = []
    monkeypatch.setattr(L, "call_with_workspace", lambda name, args, device: calls.append((name, args)))
    monkeypatch.setattr(L, "size_of", lambda name, args: 4096)
    return calls


def _turned(t):
    """t's values with its last dimension's stride the largest."""
    return t.movedim(-1, 0).contiguous().movedim(0, -1) if t.dim() > 1 else t


def _operators():
    x, g, w = _fake(3, 40, 8), _fake(5, 8), _fake(12, 8)
    ids = torch.zeros(5, dtype=torch.int64).as_subclass(type(x))
    seq = torch.zeros((3, 40), dtype=torch.int32).as_subclass(type(x))
    return {
        "recurrence": (lambda a: ops.gated_linear_recurrence(a, x, x, _fake(8), None, seq), x.clone()),
        "gated linear": (lambda a: ops.gated_linear(a, w), g.clone()),
        "loss": (lambda a: ops.linear_cross_entropy(g, a, ids), w.clone()),
    }


@pytest.mark.parametrize("name", list(_operators()))
def test_saved_tensors_at_other_strides_are_read_as_they_lie(recorded, monkeypatch, name):
    """Hooks that give back what a graph saved with other strides, or one element for all: the kernels are given rows that they
    can read, and none reads past what there is."""
    fn, leaf = _operators()[name]
    leaf.requires_grad_()
    monkeypatch.setattr(L, "device_of", lambda *ts: ts[0].device)         # (a hook's results are no fakes)
    given = []

    def one_for_all(t):
        given.append(torch.zeros((), dtype=t.dtype).expand(t.shape))
        return given[-1]

    def turned(t):
        given.append(_turned(t.detach()))
        return given[-1]

    for unpack in (one_for_all, turned):
        given.clear()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            out = fn(leaf)
        recorded.clear()
        torch.autograd.grad(out, leaf, torch.ones_like(out))
        bad = {t.data_ptr() for t in given if t.numel() > 1 and not t.is_contiguous()}
        assert bad and len(recorded) == 1
        args = recorded[0][1]
        pointers = {getattr(args, f) for f, kind in args._fields_ if kind is ctypes.c_void_p}
        assert not pointers & bad


@pytest.mark.parametrize("name", list(_operators()))
@pytest.mark.parametrize("what", ["host", "shape", "type"])
def test_saved_tensors_that_changed_are_refused(recorded, monkeypatch, name, what):
    fn, leaf = _operators()[name]
    leaf.requires_grad_()
    if what != "host":
        monkeypatch.setattr(L, "device_of", lambda *ts: ts[0].device)
    change = {"host": lambda t: t.detach().clone(), "shape": lambda t: t.detach()[..., :-1],
              "type": lambda t: t.detach().double() if t.is_floating_point() else t.detach().short()}[what]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
        out = fn(leaf)
    recorded.clear()
    with pytest.raises(ValueError, match="GPU tensors" if what == "host" else "given back as"):
        torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert not recorded
