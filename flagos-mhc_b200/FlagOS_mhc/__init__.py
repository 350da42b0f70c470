"""FlagOS_mhc on B200: the four mHC operators of liuhycs/FlagOS-mhc as
hand-written sm_100a CUDA kernels behind a C ABI (include/mhc_b200.h).

Same public names as the reference package (src/__init__.py:34-47):

    mhc_post, mhc_post_backward, mhc_pre_clamp_sinkhorn,
    mhc_pre_clamp_sinkhorn_backward          -- CUDA operators
    mhc_post_fn, mhc_pre_clamp_sinkhorn_fn,
    MhcPostFn, MhcPreClampSinkhornFn         -- autograd wrappers
    *_ref                                    -- pure-PyTorch definitions

and the operators of the sublayer between pre and post (no counterpart in the reference),
each with its ``_backward``, ``_ref``, ``_backward_ref`` and autograd wrapper:

    mhc_layer_norm                           -- layer norm
    mhc_linear                               -- matrix product + bias, activation, residual
    mhc_gated_ffn                            -- gated feed-forward block

The operators need CUDA tensors on an sm_100 GPU; there is no CPU fallback.
"""
from .mhc_post import mhc_post, mhc_post_ref
from .mhc_post_backward import mhc_post_backward, mhc_post_backward_ref
from .mhc_pre_clamp_sinkhorn import mhc_pre_clamp_sinkhorn, mhc_pre_clamp_sinkhorn_ref
from .mhc_pre_clamp_sinkhorn_backward import (mhc_pre_clamp_sinkhorn_backward,
                                              mhc_pre_clamp_sinkhorn_backward_ref)
from .mhc_layer_norm import mhc_layer_norm, mhc_layer_norm_ref
from .mhc_layer_norm_backward import mhc_layer_norm_backward, mhc_layer_norm_backward_ref
from .mhc_linear import mhc_linear, mhc_linear_ref
from .mhc_linear_backward import mhc_linear_backward, mhc_linear_backward_ref
from .mhc_gated_ffn import mhc_gated_ffn, mhc_gated_ffn_ref
from .mhc_gated_ffn_backward import mhc_gated_ffn_backward, mhc_gated_ffn_backward_ref
from .autograd import (MhcGatedFfnFn, MhcLayerNormFn, MhcLinearFn, MhcPostFn,
                       MhcPreClampSinkhornFn, mhc_gated_ffn_fn, mhc_layer_norm_fn, mhc_linear_fn,
                       mhc_post_fn, mhc_pre_clamp_sinkhorn_fn)

__all__ = [
    "mhc_post",
    "mhc_post_ref",
    "mhc_post_backward",
    "mhc_post_backward_ref",
    "mhc_pre_clamp_sinkhorn",
    "mhc_pre_clamp_sinkhorn_ref",
    "mhc_pre_clamp_sinkhorn_backward",
    "mhc_pre_clamp_sinkhorn_backward_ref",
    "MhcPostFn",
    "MhcPreClampSinkhornFn",
    "mhc_post_fn",
    "mhc_pre_clamp_sinkhorn_fn",
    "mhc_layer_norm",
    "mhc_layer_norm_ref",
    "mhc_layer_norm_backward",
    "mhc_layer_norm_backward_ref",
    "mhc_linear",
    "mhc_linear_ref",
    "mhc_linear_backward",
    "mhc_linear_backward_ref",
    "mhc_gated_ffn",
    "mhc_gated_ffn_ref",
    "mhc_gated_ffn_backward",
    "mhc_gated_ffn_backward_ref",
    "MhcLayerNormFn",
    "MhcLinearFn",
    "MhcGatedFfnFn",
    "mhc_layer_norm_fn",
    "mhc_linear_fn",
    "mhc_gated_ffn_fn",
]
