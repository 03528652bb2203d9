"""What the vocabulary's operators once answered wrongly or refused too late, as far as it shows without
a GPU."""

import ctypes
import os
import re

import pytest
import torch

from mamba2_jax import _lib as L
from mamba2_jax.models import Mamba2Config, Mamba2LMHeadModel

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(L.__file__))), "csrc")
SCORE = dict(x=4096, weight=4096, targets=4096, loss=4096, n=16, vocab=50288, dim=2560, ldx=2560, ldw=2560,
             ignore_index=-100, dtype=L.M2_BF16, target_dtype=L.M2_I64)


def score_workspace(**over):
    a = L.LinearCrossEntropyArgs(**{**SCORE, **over})
    return L.load_library().m2_linear_cross_entropy_workspace_size(ctypes.byref(a))


@pytest.mark.parametrize("n,near,far", [(16, 2560 * 1024, 2560 * 65536), (64, 2560 * 1024, 2560 * 16384),
                                        (2, 2 ** 30, 2 ** 30 + 8), (64, 2 ** 30 // 63 // 8 * 8, 2 ** 31 // 63 // 8 * 8)])
def test_far_rows_of_x_are_packed(n, near, far):
    """Few tokens are scored with x read in place, whose offsets have 32 bits; rows that lie
    further apart are packed first, into a workspace that is larger by them."""
    packed = 2 * 64 * 2560
    direct = score_workspace(n=n)
    assert score_workspace(n=n, ldx=near) == direct
    assert score_workspace(n=n, ldx=far) >= direct + packed
    assert score_workspace(n=n, ldx=2 ** 60) >= direct + packed


def test_epilogues_do_not_see_the_ring():
    """Behind the last K step no barrier says that every wavefront has read its operands, so an
    epilogue must not write to the ring that holds them: it is not given it.  (A race cannot be
    shown by running it.)"""
    with open(os.path.join(CSRC, "ce_gemm.h")) as f:
        calls = re.findall(r"epi\.template run<S>\(([^;]*)\);", f.read())
    assert len(calls) == 3 and not any("smem" in c or "lds" in c for c in calls)


def test_score_refuses_a_tied_head_that_learns():
    """Its gradient would be the head's part alone, without the embedding's.  (On the CPU: what is
    not refused is stopped by the missing GPU.)"""
    model = Mamba2LMHeadModel(Mamba2Config(d_model=64, n_layer=1, vocab_size=32, headdim=32, d_state=16))
    ids = torch.zeros((1, 4), dtype=torch.long)
    table = torch.zeros((32, 64)).requires_grad_()
    tied = {"embedding": {"weight": table}, "lm_head_weight": table}
    for head in (table, table.view(32, 64)):
        with pytest.raises(L.M2ShapeError, match="tied"):
            model.score({**tied, "lm_head_weight": head}, ids)
    own = table.detach().clone().requires_grad_()
    for params, grad in ((tied, False), ({**tied, "lm_head_weight": table.detach()}, True),
                         ({**tied, "lm_head_weight": own}, True)):
        with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="no CPU path"):
            model.score(params, ids)


@pytest.mark.parametrize("n", [20000, 2 ** 21, 2 ** 30])
def test_embedding_grad_counts_are_bounded(n):
    """The sort of many entries reads its workgroups' counts in every workgroup: there are at most 512
    of them (1 MB of counts), or the work would grow with the square of the entries."""
    a = L.EmbeddingGradArgs(n=n, vocab=2 ** 20, dim=8, ldg=8, ldo=8, padding_idx=-1, scale=1.0, id_dtype=L.M2_I64,
                            grad_dtype=L.M2_BF16, out_dtype=L.M2_F32)
    size = L.load_library().m2_embedding_grad_workspace_size(ctypes.byref(a))
    rest = 16 * n + (n // 32 + 1) * 2 * 8 * 4           # keys and places, partial rows
    assert rest <= size <= rest + 2 ** 20 + 4096


def test_embedding_grad_refuses_before_it_writes():
    """More rows than a launch takes: refused with the size, before anything is launched (a launch
    without a GPU would answer with another error)."""
    lib = L.load_library()
    a = L.EmbeddingGradArgs(ids=4096, grad=4096, out=4096, n=2 ** 31 - 5000, vocab=1000, dim=4096, ldg=4096, ldo=4096,
                            padding_idx=-1, scale=1.0, id_dtype=L.M2_I64, grad_dtype=L.M2_BF16, out_dtype=L.M2_F32,
                            workspace=4096, workspace_bytes=2 ** 62)
    assert lib.m2_embedding_grad_workspace_size(ctypes.byref(a)) == 0
    assert lib.m2_embedding_grad(ctypes.byref(a), None) == -2
    assert "too large" in lib.m2_last_error().decode()
