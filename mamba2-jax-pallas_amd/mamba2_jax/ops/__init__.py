"""mamba2_jax.ops -- the per-token ops around the SSD (HIP) and the naive SSD
formulation.

Same names as the reference's ops/__init__.py:5-15: the decode step
(selective_state_update), the depthwise causal conv before the SSD
(causal_conv1d, causal_conv1d_update) and the gated RMSNorm after it
(rms_norm_gated).  And, without counterparts there, the vocabulary's operators of training and
scoring: the loss of a linear head without its logits (linear_cross_entropy),
the embedding lookup and its gradient (embedding, embedding_grad), and the global
gradient norm (global_norm, clip_grad_norm).  And the two halves of a layer
that is trained: the gated linear recurrence over time with its gradient and its single step
(gated_linear_recurrence, gated_linear_recurrence_update), and the gated feed-forward product over
the channels with its gradient (gated_linear).
"""

from .causal_conv1d import causal_conv1d, causal_conv1d_update
from .cross_entropy import linear_cross_entropy
from .embedding import embedding, embedding_grad
from .gated_linear import gated_linear
from .gated_recurrence import gated_linear_recurrence, gated_linear_recurrence_update
from .grad_norm import clip_grad_norm, global_norm
from .rms_norm import rms_norm_gated
from .selective_state_update import selective_state_update
from .ssd_naive import mamba_chunk_scan_combined_naive

__all__ = ["selective_state_update", "mamba_chunk_scan_combined_naive", "causal_conv1d",
           "causal_conv1d_update", "rms_norm_gated", "linear_cross_entropy", "embedding",
           "embedding_grad", "clip_grad_norm", "global_norm", "gated_linear_recurrence",
           "gated_linear_recurrence_update", "gated_linear"]
