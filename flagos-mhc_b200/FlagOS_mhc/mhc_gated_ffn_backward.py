"""Backward of the gated feed-forward block on B200, and ``mhc_gated_ffn_backward_ref``."""
from __future__ import annotations

import torch

from . import _C
from .mhc_gated_ffn import _check_ffn, _kept_flag
from .mhc_linear import _act_ref, _matrix_dtype


def mhc_gated_ffn_backward(x, w_gate, w_up, w_down, gate, up, grad_y, activation="silu",
                           need_grads=(True, True, True, True)):
    """Returns (grad_x, grad_w_gate, grad_w_up, grad_w_down) in x's dtype.

    ``gate`` and ``up`` (T, F) are the forward's (``need_backward=True``), both float32 or
    both x's dtype.  One kernel
    forms grad_y w_down and, in its epilogue, the gradients of gate and up and the hidden
    product; grad_x is one product over both projections.  ``need_grads``: the outputs that
    are wanted; the others are None.
    """
    T, D, F = _check_ffn("mhc_gated_ffn_backward", x, w_gate, w_up, w_down)
    act = _C.act_code(activation)
    assert grad_y.shape == x.shape, f"grad_y shape {tuple(grad_y.shape)} != {tuple(x.shape)}"
    for name, t in (("gate", gate), ("up", up)):
        assert tuple(t.shape) == (T, F), f"{name} shape {tuple(t.shape)} != {(T, F)}"
    _C.require_cuda(x, w_gate, w_up, w_down, gate, up, grad_y)
    code = _matrix_dtype(x)
    _C.require_same("mhc_gated_ffn_backward", x, w_gate, w_up, w_down, grad_y)
    _C.require_same("mhc_gated_ffn_backward", gate, up)
    if gate.device != x.device:
        raise RuntimeError(f"FlagOS_mhc.mhc_gated_ffn_backward: tensors on {x.device} and "
                           f"{gate.device}")
    code |= _kept_flag("mhc_gated_ffn_backward", gate.dtype, x)
    need_grads = tuple(need_grads)
    if not any(need_grads):
        return (None,) * 4
    xf, xs = _C.rows(x, D)
    wg, wgs = _C.rows(w_gate, D)
    wu, wus = _C.rows(w_up, D)
    wd, wds = _C.rows(w_down, F)
    gf, gs = _C.rows(grad_y, D)
    ga, gas = _C.rows(gate, F)
    ua, uas = _C.rows(up, F)
    if gas != uas:
        ga, ua, gas = gate.contiguous(), up.contiguous(), F
    kw = dict(dtype=x.dtype, device=x.device)
    shapes = (x.shape, (F, D), (F, D), (D, F))
    outs = [torch.empty(s, **kw) if n else None for s, n in zip(shapes, need_grads)]
    L = _C.lib()
    with _C.device_guard(x.device):
        nbytes = L.mhc_gated_ffn_bwd_workspace_bytes(
            T, D, F, code, _C.unaligned((xf, xs), (wg, wgs), (wu, wus), (wd, wds), (gf, gs),
                                        *zip(outs, (D, D, D, F))))
        ws, wp = _C.workspace(nbytes, x.device)
        st = L.mhc_gated_ffn_bwd(_C.addr(xf), xs, _C.addr(wg), wgs, _C.addr(wu), wus, _C.addr(wd), wds,
                                 _C.addr(ga), _C.addr(ua), gas, _C.addr(gf), gs, T, D, F, code, act,
                                 *(_C.addr(o) for o in outs), wp, nbytes, _C.stream_addr(x.device))
    _C.check(st, "mhc_gated_ffn_backward")
    return tuple(outs)


def mhc_gated_ffn_backward_ref(x, w_gate, w_up, w_down, gate, up, grad_y, activation="silu"):
    """Pure-PyTorch definition, in fp32; any device."""
    D, dt = x.shape[-1], x.dtype
    xf, gy = x.float().reshape(-1, D), grad_y.float().reshape(-1, D)
    gh = gy @ w_down.float()
    g = gate.detach().float().requires_grad_()
    u = up.float()
    with torch.enable_grad():
        a = _act_ref(activation, g)
        gg, = torch.autograd.grad(a, g, gh * u)
    a = a.detach()
    gu = gh * a
    gx = gg @ w_gate.float() + gu @ w_up.float()
    return (gx.to(dt).reshape(x.shape), (gg.t() @ xf).to(dt), (gu.t() @ xf).to(dt),
            (gy.t() @ (a * u)).to(dt))
