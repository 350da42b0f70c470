"""torch.autograd.Function wrappers pairing each forward with its backward.

Drop-in for ``src/autograd.py`` of liuhycs/FlagOS-mhc (same classes, same
saved tensors, same defaults).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .mhc_gated_ffn import mhc_gated_ffn
from .mhc_gated_ffn_backward import mhc_gated_ffn_backward
from .mhc_layer_norm import mhc_layer_norm
from .mhc_layer_norm_backward import mhc_layer_norm_backward
from .mhc_linear import mhc_linear
from .mhc_linear_backward import mhc_linear_backward
from .mhc_post import mhc_post
from .mhc_post_backward import mhc_post_backward
from .mhc_pre_clamp_sinkhorn import mhc_pre_clamp_sinkhorn
from .mhc_pre_clamp_sinkhorn_backward import mhc_pre_clamp_sinkhorn_backward


class MhcPostFn(torch.autograd.Function):
    """src/autograd.py:14-27.  With ``next_phi`` (optional) the forward also computes the
    next layer's mix partials and appends them to ``premix_sink`` (they carry no
    gradient)."""

    @staticmethod
    def forward(ctx, x, h_res, h_out, h_post, next_phi=None, premix_sink=None):
        if next_phi is not None:
            y, pm = mhc_post(x, h_res, h_out, h_post, next_phi=next_phi.detach())
            if premix_sink is not None:
                premix_sink.append(pm)
        else:
            y = mhc_post(x, h_res, h_out, h_post)
        ctx.save_for_backward(x, h_res, h_out, h_post)
        return y

    @staticmethod
    def backward(ctx, grad_y):
        x, h_res, h_out, h_post = ctx.saved_tensors
        return mhc_post_backward(grad_y.contiguous(), x, h_res, h_out, h_post) + (None, None)


def mhc_post_fn(x, h_res, h_out, h_post, next_phi=None):
    """Autograd-aware mhc_post.

    ``next_phi`` (optional, not in the reference API): the next layer's phi; the call
    then returns ``(out, premix)`` for ``mhc_pre_clamp_sinkhorn_fn(out, next_phi, ...,
    premix=premix)`` (see :func:`FlagOS_mhc.mhc_post`).  premix carries no gradient."""
    if next_phi is None:
        return MhcPostFn.apply(x, h_res, h_out, h_post)
    sink = []
    y = MhcPostFn.apply(x, h_res, h_out, h_post, next_phi, sink)
    pm = sink[0] if sink else None
    if pm is not None:  # key it to the tensor autograd hands back
        pm._key = (y.data_ptr(), y._version, tuple(y.shape)) + pm._key[3:]
    return y, pm


class MhcPreClampSinkhornFn(torch.autograd.Function):
    """src/autograd.py:35-74: the forward runs with need_backward=True and saves
    (x, phi, alpha, base, inv_rms, x_scaled, mixes, h_res_logits, pre)."""

    @staticmethod
    def forward(ctx, x, phi, alpha, base, norm_eps, hc_eps, clamp_min, clamp_max, iter_times,
                materialize_x_scaled=True, premix=None):
        out = mhc_pre_clamp_sinkhorn(x, phi, alpha, base, norm_eps=norm_eps, hc_eps=hc_eps,
                                     clamp_min=clamp_min, clamp_max=clamp_max,
                                     iter_times=iter_times, need_backward=True,
                                     materialize_x_scaled=materialize_x_scaled, premix=premix)
        ctx.save_for_backward(x, phi, alpha, base, out["inv_rms"], out["x_scaled"],
                              out["mixes"], out["h_res_logits"], out["pre"])
        ctx.norm_eps = norm_eps
        ctx.hc_eps = hc_eps
        ctx.clamp_min = clamp_min
        ctx.clamp_max = clamp_max
        ctx.iter_times = iter_times
        return out["y"], out["post_out"], out["comb_frag"]

    @staticmethod
    def backward(ctx, grad_y, grad_post_out, grad_comb_frag):
        (x, phi, alpha, base, inv_rms, x_scaled, mixes, h_res_logits, pre) = ctx.saved_tensors
        # autograd passes None for an output that did not reach the loss
        if grad_y is None:
            grad_y = torch.zeros(x.shape[:-2] + x.shape[-1:], dtype=x.dtype, device=x.device)
        if grad_post_out is None:
            grad_post_out = torch.zeros_like(pre)
        if grad_comb_frag is None:
            grad_comb_frag = torch.zeros_like(h_res_logits)
        gx, gphi, galpha, gbase = mhc_pre_clamp_sinkhorn_backward(
            x, phi, alpha, base, inv_rms, x_scaled, mixes, h_res_logits, pre,
            grad_y.contiguous(), grad_post_out.contiguous(), grad_comb_frag.contiguous(),
            norm_eps=ctx.norm_eps, hc_eps=ctx.hc_eps, clamp_min=ctx.clamp_min,
            clamp_max=ctx.clamp_max, iter_times=ctx.iter_times)
        return (gx, gphi.to(phi.dtype), galpha.to(alpha.dtype), gbase.to(base.dtype),
                None, None, None, None, None, None, None)


def mhc_pre_clamp_sinkhorn_fn(x, phi, alpha, base, norm_eps=1e-6, hc_eps=1e-6, clamp_min=0.0,
                              clamp_max=0.0, iter_times=20, materialize_x_scaled=True,
                              premix=None):
    """Autograd-aware mhc_pre_clamp_sinkhorn. Returns (y, post_out, comb_frag).

    ``materialize_x_scaled=False`` (opt-in, not in the reference API) saves an empty
    x_scaled instead of the fp32 copy of x; the backward does not need it.
    ``premix`` (optional, not in the reference API): the mix partials that
    ``mhc_post_fn(..., next_phi=phi)`` returned with x."""
    return MhcPreClampSinkhornFn.apply(x, phi, alpha, base, norm_eps, hc_eps, clamp_min,
                                       clamp_max, iter_times, materialize_x_scaled, premix)


def _graph_wanted(*tensors):
    """Whether a call made now is differentiated later.  Asked before Function.apply, which turns
    the grad mode off around its forward."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class MhcLayerNormFn(torch.autograd.Function):
    """Layer norm; saves (x, weight, mean, rstd)."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        out = mhc_layer_norm(x, weight, bias, eps=eps, need_backward=True)
        ctx.save_for_backward(x, weight, out["mean"], out["rstd"])
        ctx.bias_dtype = bias.dtype if bias is not None else None
        return out["y"]

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        x, weight, mean, rstd = ctx.saved_tensors
        need_w, need_b = ctx.needs_input_grad[1], ctx.needs_input_grad[2]
        gx, gw, gb = mhc_layer_norm_backward(x, weight, mean, rstd, grad_y,
                                             need_param_grads=need_w or need_b)
        return (gx, gw.to(weight.dtype) if need_w else None,
                gb.to(ctx.bias_dtype) if need_b else None, None)


def mhc_layer_norm_fn(x, weight=None, bias=None, eps=1e-5):
    """Autograd-aware mhc_layer_norm. Returns y."""
    return MhcLayerNormFn.apply(x, weight, bias, eps)


class MhcLinearFn(torch.autograd.Function):
    """Linear layer; saves (x, weight, z), nothing with ``keep`` false."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, keep=True):
        out = mhc_linear(x, weight, bias=bias, residual=residual, activation=activation,
                         need_backward=keep)
        if keep:
            ctx.save_for_backward(x, weight, out["z"])
        ctx.activation = activation
        return out["y"]

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        x, weight, z = ctx.saved_tensors
        nx, nw, nb, nr = ctx.needs_input_grad[:4]
        gx, gw, gb = mhc_linear_backward(x, weight, z, grad_y, activation=ctx.activation,
                                         need_x_grad=nx, need_weight_grad=nw, need_bias_grad=nb)
        return gx, gw, gb, grad_y if nr else None, None, None


def mhc_linear_fn(x, weight, bias=None, residual=None, activation="none"):
    """Autograd-aware mhc_linear. Returns y.  z is written only if a gradient is wanted."""
    return MhcLinearFn.apply(x, weight, bias, residual, activation,
                             _graph_wanted(x, weight, bias, residual))


class MhcGatedFfnFn(torch.autograd.Function):
    """Gated feed-forward block; saves (x, w_gate, w_up, w_down, gate, up), nothing with ``keep``
    false."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation, keep=True, kept_dtype=torch.float32):
        out = mhc_gated_ffn(x, w_gate, w_up, w_down, activation=activation, need_backward=keep,
                            kept_dtype=kept_dtype)
        if keep:
            ctx.save_for_backward(x, w_gate, w_up, w_down, out["gate"], out["up"])
        ctx.activation = activation
        return out["y"]

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        return mhc_gated_ffn_backward(*ctx.saved_tensors, grad_y, activation=ctx.activation,
                                      need_grads=ctx.needs_input_grad[:4]) + (None,) * 3


def mhc_gated_ffn_fn(x, w_gate, w_up, w_down, activation="silu", kept_dtype=torch.float32):
    """Autograd-aware mhc_gated_ffn. Returns y.  gate and up are written only if a gradient is
    wanted, in ``kept_dtype`` (as in :func:`FlagOS_mhc.mhc_gated_ffn`)."""
    return MhcGatedFfnFn.apply(x, w_gate, w_up, w_down, activation,
                               _graph_wanted(x, w_gate, w_up, w_down), kept_dtype)
