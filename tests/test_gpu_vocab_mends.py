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
