"""Gated feed-forward block on B200, and its definition ``mhc_gated_ffn_ref``.

The sublayer ``h_out = F(y)`` of a hyper-connection layer.  No counterpart in the
reference.  Both projections, the activation and their product are one kernel, the down
projection a second, behind ``mhc_gated_ffn_fwd``.
"""
from __future__ import annotations

import torch

from . import _C
from .mhc_linear import _act_ref, _matrix_dtype


def _check_ffn(what, x, w_gate, w_up, w_down):
    if x.dim() not in (2, 3):
        raise ValueError(f"unsupported x.dim()={x.dim()}, expect 2 or 3")
    if w_gate.dim() != 2:
        raise ValueError(f"{what}: unsupported w_gate.dim()={w_gate.dim()}, expect 2")
    D, F = x.shape[-1], w_gate.shape[0]
    if D == 0 or F == 0:
        raise ValueError(f"{what}: empty feature dimension")
    assert tuple(w_gate.shape) == (F, D), f"w_gate shape {tuple(w_gate.shape)} != {(F, D)}"
    assert tuple(w_up.shape) == (F, D), f"w_up shape {tuple(w_up.shape)} != {(F, D)}"
    assert tuple(w_down.shape) == (D, F), f"w_down shape {tuple(w_down.shape)} != {(D, F)}"
    return x.numel() // D, D, F


def _kept_flag(what, dtype, x):
    """The entry points' flag for gate and up of this dtype."""
    if dtype == torch.float32:
        return _C.MHC_GATE_UP_F32
    if dtype != x.dtype:
        raise ValueError(f"{what}: gate and up in {dtype}; expected float32 or x's {x.dtype}")
    return 0


def mhc_gated_ffn(x, w_gate, w_up, w_down, activation="silu", need_backward=False,
                  kept_dtype=torch.float32):
    """y = (act(x w_gate^T) * (x w_up^T)) w_down^T.

    x: (T, D) or (B, S, D); w_gate, w_up: (F, D); w_down: (D, F).  All fp16 or all bf16;
    rows may be strided (the halves of one (2F, D) weight are read in place).
    ``activation`` as in :func:`FlagOS_mhc.mhc_linear`.  Products are accumulated in fp32;
    the hidden product is rounded to x's dtype, as the operand of the down projection.
    Returns a dict with ``y``; with ``need_backward=True`` also ``gate`` = x w_gate^T and
    ``up`` = x w_up^T, (T, F) in ``kept_dtype`` (the hidden product is recomputed from
    them): float32, or x's dtype, which halves what is kept and leaves gradients that are off
    by 2.1 times the rounding of the output alone in place of 1.4 times.
    """
    T, D, F = _check_ffn("mhc_gated_ffn", x, w_gate, w_up, w_down)
    act = _C.act_code(activation)
    _C.require_cuda(x, w_gate, w_up, w_down)
    code = _matrix_dtype(x)
    _C.require_same("mhc_gated_ffn", x, w_gate, w_up, w_down)
    code |= _kept_flag("mhc_gated_ffn", kept_dtype, x)
    xf, xs = _C.rows(x, D)
    gf, gs = _C.rows(w_gate, D)
    uf, us = _C.rows(w_up, D)
    df, ds = _C.rows(w_down, F)
    dev = x.device
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    gate = up = None
    ld = (F + 15) // 16 * 16  # rows start on 32-byte boundaries
    if need_backward:
        gate, up = (torch.empty(T, ld, dtype=kept_dtype, device=dev) for _ in range(2))
        if ld != F:
            gate, up = gate[:, :F], up[:, :F]
    L = _C.lib()
    with _C.device_guard(dev):
        nbytes = L.mhc_gated_ffn_fwd_workspace_bytes(
            T, D, F, code, _C.unaligned((xf, xs), (gf, gs), (uf, us), (df, ds), (y, D)))
        ws, wp = _C.workspace(nbytes, dev)
        st = L.mhc_gated_ffn_fwd(_C.addr(xf), xs, _C.addr(gf), gs, _C.addr(uf), us, _C.addr(df), ds, T,
                                 D, F, code, act, _C.addr(y), _C.addr(gate), _C.addr(up), ld, wp,
                                 nbytes, _C.stream_addr(x.device))
    _C.check(st, "mhc_gated_ffn")
    return {"y": y, "gate": gate, "up": up} if need_backward else {"y": y}


def mhc_gated_ffn_ref(x, w_gate, w_up, w_down, activation="silu"):
    """Pure-PyTorch definition, in fp32; any device."""
    xf = x.float()
    gate, up = xf @ w_gate.float().t(), xf @ w_up.float().t()
    y = (_act_ref(activation, gate) * up) @ w_down.float().t()
    F = w_gate.shape[0]
    return {"y": y.to(x.dtype), "gate": gate.reshape(-1, F), "up": up.reshape(-1, F)}
