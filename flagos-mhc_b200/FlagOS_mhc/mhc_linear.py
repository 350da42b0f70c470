"""Linear layer with bias, activation and residual in its epilogue, on B200.

The sublayer ``h_out = F(y)`` between a layer's pre and post operators.  No counterpart
in the reference.  The device work runs behind ``mhc_linear_fwd``.
"""
from __future__ import annotations

import torch

from . import _C


def _check_linear(what, x, weight, bias=None):
    if x.dim() not in (2, 3):
        raise ValueError(f"unsupported x.dim()={x.dim()}, expect 2 or 3")
    if weight.dim() != 2:
        raise ValueError(f"{what}: unsupported weight.dim()={weight.dim()}, expect 2")
    D, F = x.shape[-1], weight.shape[0]
    if D == 0 or F == 0:
        raise ValueError(f"{what}: empty feature dimension")
    assert weight.shape[1] == D, f"weight shape {tuple(weight.shape)} != {(F, D)}"
    if bias is not None:
        assert tuple(bias.shape) == (F,), f"bias shape {tuple(bias.shape)} != {(F,)}"
    return x.numel() // D, D, F


def _matrix_dtype(x):
    """The matrix products take fp16 and bf16."""
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"FlagOS_mhc: unsupported dtype {x.dtype}; expected float16/bfloat16")
    return _C.dtype_code(x.dtype)


def mhc_linear(x, weight, bias=None, residual=None, activation="none", need_backward=False):
    """y = act(x weight^T + bias) + residual.

    x: (T, D) or (B, S, D); weight: (F, D); bias: (F,); residual: x's leading shape + (F,).
    All fp16 or all bf16; rows may be strided.  ``activation``: "none", "relu", "gelu"
    (by erf), "gelu_tanh" or "silu".  Products are accumulated in fp32, the epilogue runs
    in fp32 and y is rounded once.  Returns a dict with ``y``; with ``need_backward=True``
    also ``z`` = x weight^T + bias in x's dtype, which the backward of the activation reads
    (None for "none").
    """
    T, D, F = _check_linear("mhc_linear", x, weight, bias)
    act = _C.act_code(activation)
    out_shape = x.shape[:-1] + (F,)
    if residual is not None:
        assert residual.shape == out_shape, \
            f"residual shape {tuple(residual.shape)} != {tuple(out_shape)}"
    _C.require_cuda(x, weight, bias, residual)
    code = _matrix_dtype(x)
    _C.require_same("mhc_linear", x, weight, bias, residual)
    xf, xs = _C.rows(x, D)
    wf, wstr = _C.rows(weight, D)
    rf, rs = _C.rows(residual, F) if residual is not None else (None, 0)
    bf = bias
    if bf is not None and (not bf.is_contiguous() or bf.data_ptr() & 31):
        bf = bf.clone(memory_format=torch.contiguous_format)  # the epilogue reads it in packs
    dev = x.device
    y = torch.empty(out_shape, dtype=x.dtype, device=dev)
    z = torch.empty(out_shape, dtype=x.dtype, device=dev) if need_backward and act else None
    L = _C.lib()
    with _C.device_guard(dev):
        nbytes = L.mhc_linear_fwd_workspace_bytes(T, D, F, code,
                                                  _C.unaligned((xf, xs), (wf, wstr), (rf, rs), (y, F)))
        ws, wp = _C.workspace(nbytes, dev)
        st = L.mhc_linear_fwd(_C.addr(xf), xs, _C.addr(wf), wstr, _C.addr(bf), _C.addr(rf), rs, T, D,
                              F, code, act, _C.addr(y), _C.addr(z), wp, nbytes, _C.stream_addr(x.device))
    _C.check(st, "mhc_linear")
    return {"y": y, "z": z} if need_backward else {"y": y}


def _act_ref(name, z):
    Fn = torch.nn.functional
    return {"none": lambda v: v, "relu": torch.relu, "gelu": Fn.gelu,
            "gelu_tanh": lambda v: Fn.gelu(v, approximate="tanh"), "silu": Fn.silu}[name](z)


def mhc_linear_ref(x, weight, bias=None, residual=None, activation="none"):
    """Pure-PyTorch definition, in fp32; any device."""
    z = x.float() @ weight.float().t()
    if bias is not None:
        z = z + bias.float()
    y = _act_ref(activation, z)
    if residual is not None:
        y = y + residual.float()
    return {"y": y.to(x.dtype), "z": None if activation == "none" else z.to(x.dtype)}
