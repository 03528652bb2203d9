"""mamba2_jax.ops -- the per-token ops around the SSD (HIP) and the naive SSD
formulation.

Same names as the reference's ops/__init__.py:5-15: the decode step
(selective_state_update), the depthwise causal conv before the SSD
(causal_conv1d, causal_conv1d_update) and the gated RMSNorm after it
(rms_norm_gated).  And, without counterparts there, the vocabulary's operators of training and
scoring: the loss of a linear head without its logits (linear_cross_entropy),
the embedding lookup and its gradient (embedding, embedding_grad), and the global
gradient norm (global_norm, clip_grad_norm).
"""

from .causal_conv1d import causal_conv1d, causal_conv1d_update
from .cross_entropy import linear_cross_entropy
from .embedding import embedding, embedding_grad
from .grad_norm import clip_grad_norm, global_norm
from .rms_norm import rms_norm_gated
from .selective_state_update import selective_state_update
from .ssd_naive import mamba_chunk_scan_combined_naive

__all__ = ["selective_state_update", "mamba_chunk_scan_combined_naive", "causal_conv1d",
           "causal_conv1d_update", "rms_norm_gated", "linear_cross_entropy", "embedding",
           "embedding_grad", "clip_grad_norm", "global_norm"]
