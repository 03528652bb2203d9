"""What the vocabulary's operators once answered wrongly.  Formulas and tolerances are those of
test_gpu_vocab."""

import pytest
import torch

from gpu_util import announce
from mamba2_jax import ops
from test_gpu_vocab import DEV, DT, IGN, Ref, ce_inputs, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,apart", [(16, 150_000_000), (40, 60_000_000), (64, 34_100_000)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_score_rows_far_apart(n, apart, dtype):
    """The last positions of long prompts: rows of x whose offsets pass 32 bits, as those rows
    beside each other."""
    announce("rows far apart", n, apart, dtype)
    x, w, t = ce_inputs(n, 700, 128, dtype, 0.2, key=50)
    flat = torch.empty(((n - 1) * apart + 128,), device=DEV, dtype=DT[dtype])
    far = flat.as_strided((n, 128), (apart, 1))
    far.copy_(x)
    assert (n - 1) * apart * x.element_size() > 2 ** 32
    r = Ref(x, w, t, torch.ones(n, device=DEV, dtype=torch.float64))
    loss = ops.linear_cross_entropy(far, w, t, reduction="none")
    within(loss, r.loss, r.loss_tol, "loss")
    assert not bool(loss[t == IGN].any())


@pytest.mark.parametrize("n", [1, 16, 17, 64])
@pytest.mark.parametrize("dim", [64, 192, 256, 320, 448, 576, 832, 2560])
def test_score_last_step_in_each_slot(n, dim):
    """Few tokens: the wavefronts of a tile put their sums together in LDS that no operand lies in,
    whichever slot of the ring (of four up to 16 tokens, of three beyond) the last K step
    is in.  16 runs of more tiles than the card has CUs, equal to the bit."""
    announce("last step in each slot", n, dim)
    x, w, t = ce_inputs(n, 128 * 300, dim, "bf16", key=51)
    r = Ref(x, w, t, torch.ones(n, device=DEV, dtype=torch.float64))
    loss = ops.linear_cross_entropy(x, w, t, reduction="none")
    within(loss, r.loss, r.loss_tol, "loss")
    for _ in range(15):
        assert torch.equal(ops.linear_cross_entropy(x, w, t, reduction="none"), loss)
