"""The operators of a trained layer where they are used together (examples/gated_layers.py): a training step, whole
and operator by operator; a captured one; and a prompt followed by single tokens."""

import os
import sys

import pytest
import torch

from gpu_util import announce
from mamba2_jax import ops

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import gated_layers as M  # noqa: E402

pytestmark = pytest.mark.gpu


def text(vocab, batch, seqlen, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, vocab, (batch, seqlen + 1), generator=g, device="cuda")


def packed(batch, seqlen):
    """Two documents in each row, padding behind the second."""
    seq = torch.zeros((batch, seqlen), dtype=torch.int32, device="cuda")
    seq[:, seqlen // 3:] = 1
    seq[:, seqlen - seqlen // 8:] = -1
    return seq


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("docs", [False, True])
def test_step_whole_and_in_parts(dtype, docs):
    """The gradients of one graph equal, bit for bit, those of the operators' own graphs chained by hand."""
    announce("layer step", dtype, docs)
    vocab, dim, hidden, batch, n = 97, 72, 100, 2, 150
    params = M.init(vocab, dim, hidden, 2, dtype)
    ids = text(vocab, batch, n, 5)
    seq = packed(batch, n) if docs else None
    targets = ids[:, 1:].clone()
    if docs:
        targets[seq < 0] = -100
    loss = M.loss_of(params, ids[:, :-1], targets, seq)
    whole = torch.autograd.grad(loss, M.leaves(params))
    # forward, each operator on detached inputs
    cut = lambda t: t.detach().requires_grad_()
    u = ops.embedding(ids[:, :-1], params["embedding"])
    first, tape = u, []
    for b in params["blocks"]:
        ui = cut(u)
        proj = ui @ b["w_in"]
        x, r, i = (cut(t) for t in proj.detach().chunk(3, dim=-1))
        A = -torch.exp(b["A_log"])
        Ai = cut(A)
        h, _ = ops.gated_linear_recurrence(x, r, i, Ai, seq_idx=seq, return_final_states=True)
        hi = cut(h)
        um = cut(ui.detach() + hi @ b["w_out"])
        up = ops.gated_linear(um, b["w_up"])
        upi = cut(up)
        tape.append((b, ui, proj, A, (x, r, i, Ai), h, hi, hi @ b["w_out"], um, up, upi, upi @ b["w_down"]))
        u = um.detach() + tape[-1][-1].detach()
    ul = cut(u)
    l2 = ops.linear_cross_entropy(ul, params["head"], targets)
    assert torch.equal(l2, loss)
    du, dhead = torch.autograd.grad(l2, (ul, params["head"]))
    grads = []
    for b, ui, proj, A, xria, h, hi, out, um, up, upi, down in reversed(tape):
        dup, dwd = torch.autograd.grad(down, (upi, b["w_down"]), du)
        dum, dwu = torch.autograd.grad(up, (um, b["w_up"]), dup)
        du = du + dum
        dh, dwo = torch.autograd.grad(out, (hi, b["w_out"]), du)
        *dxri, dA = torch.autograd.grad(h, xria, dh)
        (dA,) = torch.autograd.grad(A, b["A_log"], dA)
        dui, dwi = torch.autograd.grad(proj, (ui, b["w_in"]), torch.cat(dxri, dim=-1))
        du = du + dui
        grads = [dwi, dA, dwo, dwu, dwd, *grads]
    (de,) = torch.autograd.grad(first, params["embedding"], du)
    names = ["embedding", *[f"{k}{j}" for j in range(2) for k in params["blocks"][0]], "head"]
    for name, p, q in zip(names, whole, [de, *grads, dhead]):
        assert torch.equal(p, q), name
        assert bool(p.isfinite().all()) and float(p.float().abs().max()) > 0


def test_documents_do_not_meet():
    """Packed documents give the losses that they give by themselves, whatever stands behind the last."""
    announce("documents")
    vocab, dim, n = 97, 64, 180
    params = M.init(vocab, dim, 96, 2, torch.float32)
    ids = text(vocab, 1, n, 6)
    seq = packed(1, n)
    per = lambda i, s: ops.linear_cross_entropy(M.layer(M.layer(ops.embedding(i, params["embedding"]), params["blocks"][0],
                                                               seq_idx=s)[0], params["blocks"][1], seq_idx=s)[0],
                                                params["head"], i, reduction="none")
    with torch.no_grad():
        whole = per(ids[:, :n], seq)
        a, b = n // 3, n - n // 8
        one, two = per(ids[:, :a], None), per(ids[:, a:b], None)
    # (the same sums but for where the joins of maps and the tiles of the products fall: float32 roundings, which
    # four products of 64 to 96 terms and 120 steps of the recurrence, of magnitudes up to 30, carry to the loss)
    tol = 30 * (4 * 40 + 120) * 2.0 ** -24 * 4
    assert float((whole[:, :a] - one).abs().max()) <= tol
    assert float((whole[:, a:b] - two).abs().max()) <= tol


def test_captured_step():
    """A captured training step gives on every replay the eager step's gradients."""
    announce("captured step")
    vocab, dim, batch, n = 97, 64, 2, 140
    params = M.init(vocab, dim, 96, 2)
    ids = text(vocab, batch, n, 7)
    buf = ids.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(M.loss_of(params, buf[:, :-1], buf[:, 1:]), M.leaves(params))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = M.loss_of(params, buf[:, :-1], buf[:, 1:])
        grads = torch.autograd.grad(loss, M.leaves(params))
    for k in range(4):
        other = text(vocab, batch, n, 20 + k)
        buf.copy_(other)
        graph.replay()
        torch.cuda.synchronize()
        l2 = M.loss_of(params, other[:, :-1], other[:, 1:])
        want = torch.autograd.grad(l2, M.leaves(params))
        assert torch.equal(loss, l2)
        assert all(torch.equal(p, q) for p, q in zip(grads, want))


def test_two_streams_at_once():
    """Training steps of two models that run beside each other on two streams, replayed from two graphs too: each as alone."""
    announce("two streams")
    sets = [(M.init(53, 64, 96, 2), text(53, 2, 150, 1)), (M.init(61, 128, 72, 1), text(61, 1, 700, 2))]
    run = lambda p, ids: [*torch.autograd.grad(M.loss_of(p, ids[:, :-1], ids[:, 1:]), M.leaves(p))]
    want = [run(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(run(*sets[k]))
    torch.cuda.synchronize()
    graphs = []
    for k in (0, 1):
        graphs.append((torch.cuda.CUDAGraph(), []))
        with torch.cuda.graph(graphs[k][0], stream=streams[k]):
            graphs[k][1].extend(run(*sets[k]))
    for _ in range(3):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                graphs[k][0].replay()
    torch.cuda.synchronize()
    for k in (0, 1):
        for one in (*got[k], graphs[k][1]):
            assert all(torch.equal(p, q) for p, q in zip(one, want[k]))


def test_prompt_then_tokens():
    """A prompt in one call and the tokens behind it one by one: the states and outputs of the whole in one call."""
    announce("prompt then tokens")
    dim, n, more = 64, 130, 7
    b = M.init(31, dim, 96, 1, torch.float32)["blocks"][0]
    g = torch.Generator(device="cuda").manual_seed(9)
    u = torch.randn((3, n + more, dim), generator=g, device="cuda")
    with torch.no_grad():
        whole, last = M.layer(u, b)
        got, state = M.layer(u[:, :n], b)
        tol = 400 * 2.0 ** -24 * float(whole.abs().max())     # sums of up to 96 terms in another order, twice
        assert float((got - whole[:, :n]).abs().max()) <= tol
        for t in range(n, n + more):
            y = M.layer_step(u[:, t], b, state)
            assert float((y - whole[:, t]).abs().max()) <= tol
        assert float((state - last).abs().max()) <= tol


def test_example_runs():
    announce("example")
    params = M.init(50, 64, 96, 2)
    ids = text(50, 2, 90, 3)
    for _ in range(2):
        loss, norm = M.step(params, ids[:, :-1], ids[:, 1:])
        assert bool(loss.isfinite()) and bool(norm.isfinite())
