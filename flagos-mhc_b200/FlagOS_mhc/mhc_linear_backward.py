"""Backward of the linear layer on B200, and ``mhc_linear_backward_ref``."""
from __future__ import annotations

import torch

from . import _C
from .mhc_linear import _act_ref, _check_linear, _matrix_dtype


def mhc_linear_backward(x, weight, z, grad_y, activation="none", need_x_grad=True,
                        need_weight_grad=True, need_bias_grad=True):
    """Returns (grad_x, grad_weight, grad_bias), each in x's dtype or None if not needed.

    ``z`` is the forward's (None for activation "none").  gz = grad_y * act'(z);
    grad_x = gz weight, grad_weight = gz^T x, grad_bias = sum of gz over the tokens in a
    fixed order.  The gradient of the forward's residual is grad_y itself.
    """
    T, D, F = _check_linear("mhc_linear_backward", x, weight)
    act = _C.act_code(activation)
    assert grad_y.shape == x.shape[:-1] + (F,), \
        f"grad_y shape {tuple(grad_y.shape)} != {tuple(x.shape[:-1] + (F,))}"
    if act:
        if z is None:
            raise ValueError(f"mhc_linear_backward: activation {activation!r} needs the "
                             "forward's z (need_backward=True)")
        assert z.shape == grad_y.shape, f"z shape {tuple(z.shape)} != {tuple(grad_y.shape)}"
    else:
        z = None
    _C.require_cuda(x, weight, z, grad_y)
    code = _matrix_dtype(x)
    _C.require_same("mhc_linear_backward", x, weight, z, grad_y)
    if not (need_x_grad or need_weight_grad or need_bias_grad):
        return (None,) * 3
    xf, xs = _C.rows(x, D)
    wf, wstr = _C.rows(weight, D)
    gf, gs = _C.rows(grad_y, F)
    zf, zs = _C.rows(z, F) if z is not None else (None, 0)
    kw = dict(dtype=x.dtype, device=x.device)
    gx = torch.empty(x.shape, **kw) if need_x_grad else None
    gw = torch.empty(F, D, **kw) if need_weight_grad else None
    gb = torch.empty(F, **kw) if need_bias_grad else None
    L = _C.lib()
    with _C.device_guard(x.device):
        nbytes = L.mhc_linear_bwd_workspace_bytes(
            T, D, F, code, act, _C.unaligned((xf, xs), (wf, wstr), (gf, gs), (gx, D), (gw, D)))
        ws, wp = _C.workspace(nbytes, x.device)
        st = L.mhc_linear_bwd(_C.addr(xf), xs, _C.addr(wf), wstr, _C.addr(zf), zs, _C.addr(gf), gs, T,
                              D, F, code, act, _C.addr(gx), _C.addr(gw), _C.addr(gb), wp, nbytes,
                              _C.stream_addr(x.device))
    _C.check(st, "mhc_linear_backward")
    return gx, gw, gb


def mhc_linear_backward_ref(x, weight, z, grad_y, activation="none"):
    """Pure-PyTorch definition, in fp32; any device."""
    D, F = x.shape[-1], weight.shape[0]
    gz = grad_y.float().reshape(-1, F)
    if activation != "none":
        zf = z.detach().float().reshape(-1, F).requires_grad_()
        with torch.enable_grad():
            gz, = torch.autograd.grad(_act_ref(activation, zf), zf, gz)
    gx = (gz @ weight.float()).to(x.dtype).reshape(x.shape)
    gw = (gz.t() @ x.float().reshape(-1, D)).to(x.dtype)
    return gx, gw, gz.sum(0).to(x.dtype)
