"""Layer norm forward on B200, and its pure-PyTorch definition ``mhc_layer_norm_ref``.

The norm between a layer's pre operator (its ``y``) and the sublayer.  No counterpart in
the reference.  The device work is one CUDA kernel behind ``mhc_layer_norm_fwd``.
"""
from __future__ import annotations

import torch

from . import _C


def _check_params(x, weight, bias):
    if x.dim() not in (2, 3):
        raise ValueError(f"unsupported x.dim()={x.dim()}, expect 2 or 3")
    D = x.shape[-1]
    if D == 0:
        raise ValueError("mhc_layer_norm: rows of width 0")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            assert p.dim() == 1 and p.numel() == D, f"{name} shape {tuple(p.shape)} != {(D,)}"
            if p.device != x.device:
                raise RuntimeError(f"FlagOS_mhc.mhc_layer_norm: tensors on {x.device} and "
                                   f"{p.device}")
    return D


def _param(p):
    """A parameter as the kernels take it: packed fp32."""
    if p is None or (p.dtype == torch.float32 and p.is_contiguous()):
        return p
    return p.to(torch.float32).contiguous()


def mhc_layer_norm(x, weight=None, bias=None, eps=1e-5, need_backward=False):
    """y = (x - mean) * rstd * weight + bias over the last dimension.

    x: (T, D) or (B, S, D), fp32 / fp16 / bf16, rows may be strided.  ``weight`` and
    ``bias`` (D,) of any float dtype, used in fp32; None is 1 and 0.  mean and
    rstd = 1 / sqrt(variance + eps) are computed in fp32, the variance from the centred
    values.  Returns a dict with ``y`` (x's shape and dtype); with ``need_backward=True``
    also ``mean`` and ``rstd`` (T,) fp32.
    """
    D = _check_params(x, weight, bias)
    if not eps >= 0.0:
        raise ValueError(f"mhc_layer_norm: eps={eps}")
    _C.require_cuda(x, weight, bias)
    code = _C.dtype_code(x.dtype)
    T = x.numel() // D
    xf, xs = _C.rows(x, D)
    w, b = _param(weight), _param(bias)
    dev = x.device
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean = rstd = None
    if need_backward:
        mean = torch.empty(T, dtype=torch.float32, device=dev)
        rstd = torch.empty(T, dtype=torch.float32, device=dev)
    with _C.device_guard(dev):
        st = _C.lib().mhc_layer_norm_fwd(_C.addr(xf), xs, _C.addr(w), _C.addr(b), T, D, code,
                                         float(eps), _C.addr(y), _C.addr(mean), _C.addr(rstd),
                                         _C.stream_addr(x.device))
    _C.check(st, "mhc_layer_norm")
    return {"y": y, "mean": mean, "rstd": rstd} if need_backward else {"y": y}


def mhc_layer_norm_ref(x, weight=None, bias=None, eps=1e-5):
    """Pure-PyTorch definition; any device.  Returns the dict of ``need_backward=True``."""
    xf = x.float().reshape(-1, x.shape[-1])
    mean = xf.mean(-1)
    c = xf - mean[:, None]
    rstd = (c.pow(2).mean(-1) + eps).rsqrt()
    y = c * rstd[:, None]
    if weight is not None:
        y = y * weight.float()
    if bias is not None:
        y = y + bias.float()
    return {"y": y.to(x.dtype).reshape(x.shape), "mean": mean, "rstd": rstd}
