"""Layer norm backward on B200, and ``mhc_layer_norm_backward_ref``."""
from __future__ import annotations

import torch

from . import _C
from .mhc_layer_norm import _check_params, _param


def mhc_layer_norm_backward(x, weight, mean, rstd, grad_y, need_param_grads=True):
    """Returns (grad_x, grad_weight, grad_bias).

    ``mean`` and ``rstd`` (T,) are the forward's (``need_backward=True``).  grad_x has x's
    shape and dtype; grad_weight and grad_bias are (D,) fp32 views of one buffer (one
    collective), summed over the tokens in a fixed order, or None with
    ``need_param_grads=False``.
    """
    D = _check_params(x, weight, None)
    T = x.numel() // D
    assert grad_y.shape == x.shape, f"grad_y shape {tuple(grad_y.shape)} != {tuple(x.shape)}"
    for name, p in (("mean", mean), ("rstd", rstd)):
        assert p.numel() == T, f"{name} has {p.numel()} values, expect {T}"
    _C.require_cuda(x, weight, mean, rstd, grad_y)
    _C.require_same("mhc_layer_norm_backward", x, grad_y)
    _C.require_same("mhc_layer_norm_backward", mean, rstd)
    if mean.device != x.device:
        raise RuntimeError(f"FlagOS_mhc.mhc_layer_norm_backward: tensors on {x.device} and "
                           f"{mean.device}")
    code = _C.dtype_code(x.dtype)
    xf, xs = _C.rows(x, D)
    gf, gs = _C.rows(grad_y, D)
    w, m, r = _param(weight), _param(mean), _param(rstd)
    dev = x.device
    grad_x = torch.empty_like(x, memory_format=torch.contiguous_format)
    gw = gb = ws = wp = None
    nbytes = 0
    L = _C.lib()
    with _C.device_guard(dev):
        if need_param_grads:
            gw, gb = torch.empty(2, D, dtype=torch.float32, device=dev).unbind(0)
            nbytes = L.mhc_layer_norm_bwd_workspace_bytes(T, D, code)
            ws, wp = _C.workspace(nbytes, dev)
        st = L.mhc_layer_norm_bwd(_C.addr(xf), xs, _C.addr(w), _C.addr(m), _C.addr(r), _C.addr(gf), gs,
                                  T, D, code, _C.addr(grad_x), _C.addr(gw), _C.addr(gb), wp, nbytes,
                                  _C.stream_addr(x.device))
    _C.check(st, "mhc_layer_norm_backward")
    return grad_x, gw, gb


def mhc_layer_norm_backward_ref(x, weight, mean, rstd, grad_y):
    """Pure-PyTorch definition; any device."""
    D = x.shape[-1]
    xf, gy = x.float().reshape(-1, D), grad_y.float().reshape(-1, D)
    xh = (xf - mean.reshape(-1, 1)) * rstd.reshape(-1, 1)
    h = gy * weight.float() if weight is not None else gy
    gx = rstd.reshape(-1, 1) * (h - h.mean(-1, keepdim=True) - xh * (h * xh).mean(-1, keepdim=True))
    return gx.to(x.dtype).reshape(x.shape), (gy * xh).sum(0), gy.sum(0)
