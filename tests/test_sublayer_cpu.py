"""The sublayer operators without a GPU: refusals (Python and C ABI), workspace sizes, and
the pure-PyTorch ``*_ref`` functions against the float64 oracle."""
import ctypes

import pytest
import torch

import FlagOS_mhc as M
from FlagOS_mhc import _C
from oracle import sublayer_oracle as S

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
P = ctypes.c_void_p(4096)


def r(*shape, dt=torch.bfloat16):
    return torch.randn(*shape).to(dt)


def test_cpu_tensors_are_refused():
    x, w = r(4, 16), r(8, 16)
    for call in (lambda: M.mhc_layer_norm(x), lambda: M.mhc_linear(x, w),
                 lambda: M.mhc_gated_ffn(x, w, w, w.t().contiguous()),
                 lambda: M.mhc_layer_norm_backward(x, None, r(4), r(4), x),
                 lambda: M.mhc_linear_backward(x, w, None, r(4, 8)),
                 lambda: M.mhc_gated_ffn_backward(x, w, w, w.t().contiguous(), r(4, 8), r(4, 8), x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_shapes_and_names_are_checked_first():
    x, w = r(4, 16), r(8, 16)
    wd = w.t().contiguous()
    with pytest.raises(ValueError):
        M.mhc_layer_norm(r(16))
    with pytest.raises(ValueError):
        M.mhc_layer_norm(r(2, 2, 4, 16))
    with pytest.raises(ValueError):
        M.mhc_layer_norm(r(4, 0))
    with pytest.raises(AssertionError):
        M.mhc_layer_norm(x, r(15))
    with pytest.raises(AssertionError):
        M.mhc_layer_norm(x, r(16), r(16, 1))
    with pytest.raises(ValueError):
        M.mhc_layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError):
        M.mhc_layer_norm(x, eps=float("nan"))
    with pytest.raises(AssertionError):
        M.mhc_layer_norm_backward(x, None, r(4), r(4), r(4, 15))
    with pytest.raises(AssertionError):
        M.mhc_layer_norm_backward(x, None, r(3), r(4), x)
    with pytest.raises(ValueError):
        M.mhc_linear(r(16), w)
    with pytest.raises(ValueError):
        M.mhc_linear(x, r(16))
    with pytest.raises(AssertionError):
        M.mhc_linear(x, r(8, 15))
    with pytest.raises(ValueError):
        M.mhc_linear(x, r(0, 16))
    with pytest.raises(AssertionError):
        M.mhc_linear(x, w, bias=r(7))
    with pytest.raises(AssertionError):
        M.mhc_linear(x, w, residual=r(4, 16))
    with pytest.raises(ValueError, match="activation"):
        M.mhc_linear(x, w, activation="swish")
    with pytest.raises(ValueError, match="need_backward"):
        M.mhc_linear_backward(x, w, None, r(4, 8), activation="silu")
    with pytest.raises(AssertionError):
        M.mhc_linear_backward(x, w, r(4, 7), r(4, 8), activation="silu")
    with pytest.raises(AssertionError):
        M.mhc_linear_backward(x, w, None, r(4, 16))
    with pytest.raises(ValueError):
        M.mhc_gated_ffn(r(16), w, w, wd)
    with pytest.raises(AssertionError):
        M.mhc_gated_ffn(x, w, r(9, 16), wd)
    with pytest.raises(AssertionError):
        M.mhc_gated_ffn(x, w, w, w)
    with pytest.raises(ValueError, match="activation"):
        M.mhc_gated_ffn(x, w, w, wd, activation=None)
    with pytest.raises(AssertionError):
        M.mhc_gated_ffn_backward(x, w, w, wd, r(4, 9), r(4, 8), x)
    with pytest.raises(AssertionError):
        M.mhc_gated_ffn_backward(x, w, w, wd, r(4, 8), r(4, 8), r(4, 8))


def test_devices_and_dtypes_of_one_call():
    x = torch.empty(2, 3, device="meta", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="meta"):
        _C.require_same("op", r(2, 3), x)
    with pytest.raises(ValueError, match="dtypes"):
        _C.require_same("op", r(2, 3), r(2, 3, dt=torch.float16))
    _C.require_same("op", r(2, 3), None, r(5))


def test_c_abi_refusals():
    L = _C.lib()
    inv, dty, wsp = _C.MHC_ERR_INVALID_ARGUMENT, _C.MHC_ERR_UNSUPPORTED_DTYPE, _C.MHC_ERR_WORKSPACE

    def ln(x=P, xs=16, T=4, D=16, dt=2, eps=1e-5, y=P):
        return L.mhc_layer_norm_fwd(x, xs, None, None, T, D, dt, eps, y, None, None, None)

    assert ln(T=-1) == inv and ln(D=0) == inv and ln(xs=15) == inv and ln(eps=-1.0) == inv
    assert ln(eps=float("nan")) == inv and ln(dt=3) == dty and ln(x=None) == inv
    assert ln(y=None) == inv and ln(T=0, x=None, y=None) == _C.MHC_OK

    def lnb(T=4, D=16, gw=P, gb=P, ws=P, nb=1 << 20, mean=P):
        return L.mhc_layer_norm_bwd(P, 16, None, mean, P, P, 16, T, D, 2, P, gw, gb, ws, nb, None)

    assert lnb(gb=None) == inv and lnb(mean=None) == inv
    assert lnb(ws=None) == wsp and lnb(nb=8) == wsp and lnb(ws=ctypes.c_void_p(4100)) == wsp
    assert lnb(T=0, gw=None, gb=None) == _C.MHC_OK

    def lin(xs=16, wstr=16, res=None, rs=0, T=4, D=16, F=8, dt=2, act=0, y=P):
        return L.mhc_linear_fwd(P, xs, P, wstr, None, res, rs, T, D, F, dt, act, y, None, None, 0,
                                None)

    assert lin(xs=15) == inv and lin(wstr=15) == inv and lin(res=P, rs=7) == inv
    assert lin(T=-1) == inv and lin(D=0) == inv and lin(F=0) == inv and lin(y=None) == inv
    assert lin(dt=0) == dty and lin(act=5) == inv and lin(act=-1) == inv
    assert lin(T=0, y=None) == _C.MHC_OK
    assert lin(T=2 ** 31) == inv and lin(D=2 ** 31, xs=2 ** 31, wstr=2 ** 31) == inv

    def linb(z=P, zs=8, act=4, ws=P, nb=1 << 30, dt=2, gs=8):
        return L.mhc_linear_bwd(P, 16, P, 16, z, zs, P, gs, 4, 16, 8, dt, act, P, P, P, ws, nb, None)

    assert linb(z=None) == inv and linb(zs=7) == inv and linb(gs=7) == inv and linb(dt=0) == dty
    assert linb(ws=None) == wsp and linb(nb=1) == wsp

    def ffn(gate=None, up=None, gs=0, ws=P, nb=1 << 30, dt=2, act=4, wds=8):
        return L.mhc_gated_ffn_fwd(P, 16, P, 16, P, 16, P, wds, 4, 16, 8, dt, act, P, gate, up, gs,
                                   ws, nb, None)

    assert ffn(gate=P) == inv and ffn(gate=P, up=P, gs=7) == inv and ffn(dt=0) == dty
    assert ffn(wds=7) == inv and ffn(act=9) == inv and ffn(ws=None) == wsp and ffn(nb=1) == wsp

    def ffnb(gate=P, gs=8, gys=16, ws=P, nb=1 << 30):
        return L.mhc_gated_ffn_bwd(P, 16, P, 16, P, 16, P, 8, gate, P, gs, P, gys, 4, 16, 8, 2, 4,
                                   P, P, P, P, ws, nb, None)

    assert ffnb(gate=None) == inv and ffnb(gs=7) == inv and ffnb(gys=15) == inv
    assert ffnb(ws=None) == wsp and ffnb(nb=1) == wsp


def test_sublayer_workspace_sizes():
    L = _C.lib()
    assert L.mhc_layer_norm_bwd_workspace_bytes(4096, 1024, 2) >= 2 * 1024 * 4
    assert L.mhc_layer_norm_bwd_workspace_bytes(4096, 0, 2) == 0
    # h; gg, gu and h
    assert L.mhc_gated_ffn_fwd_workspace_bytes(100, 64, 72, 2, 0) >= 100 * 72 * 2
    assert L.mhc_gated_ffn_bwd_workspace_bytes(100, 64, 72, 2, 0) >= 3 * 100 * 72 * 2
    assert L.mhc_gated_ffn_bwd_workspace_bytes(100, 64, 72, 0, 0) == 0
    assert L.mhc_linear_bwd_workspace_bytes(100, 64, 72, 2, 4, 0) >= 100 * 72 * 2
    for f, a in ((L.mhc_linear_fwd_workspace_bytes, (100, 65, 72, 2)),
                 (L.mhc_linear_bwd_workspace_bytes, (100, 65, 72, 2, 4)),
                 (L.mhc_gated_ffn_fwd_workspace_bytes, (100, 65, 72, 2)),
                 (L.mhc_gated_ffn_bwd_workspace_bytes, (100, 65, 72, 2))):
        assert f(*a, 1) >= f(*a, 0)


def test_row_views():
    x = r(6, 40)
    assert _C.rows(x[:, :16], 16)[1] == 40
    assert _C.rows(x[:, :16], 16)[0].data_ptr() == x.data_ptr()
    t, ts = _C.rows(x.t(), 6)          # not row-contiguous: packed
    assert ts == 6 and t.is_contiguous()
    assert _C.rows(x[:1].expand(5, 40), 40)[1] == 40
    assert _C.unaligned((x, 40)) == 0 and _C.unaligned((x, 41)) == 1
    assert _C.unaligned((x, 40), (x[:, 1:], 40)) == 1


@pytest.mark.parametrize("name", ACTS)
def test_refs_match_the_oracle(name):
    f32 = torch.float32
    g = torch.Generator().manual_seed(3)

    def n(*shape):
        return torch.randn(*shape, generator=g)

    def close(a, b):
        assert a.dtype == f32 and torch.allclose(a.double(), b, rtol=2e-5, atol=2e-5)

    x, w, b, res, gy = n(9, 12), n(7, 12), n(7), n(9, 7), n(9, 7)
    o = M.mhc_linear_ref(x, w, b, res, name)
    y, z = S.linear(x, w, b, res, name)
    close(o["y"], y)
    for a, c in zip(M.mhc_linear_backward_ref(x, w, z.float(), gy, name),
                    S.linear_bwd(x, w, z, gy, name)):
        close(a, c)
    wu, wd, gx = n(7, 12), n(12, 7), n(9, 12)
    o = M.mhc_gated_ffn_ref(x, w, wu, wd, name)
    y, gate, up = S.gated_ffn(x, w, wu, wd, name)
    close(o["y"], y)
    for a, c in zip(M.mhc_gated_ffn_backward_ref(x, w, wu, wd, gate.float(), up.float(), gx, name),
                    S.gated_ffn_bwd(x, w, wu, wd, gate, up, gx, name)):
        close(a, c)
    lw, lb = n(12), n(12)
    o = M.mhc_layer_norm_ref(x, lw, lb, 1e-5)
    y, mean, rstd = S.layer_norm(x, lw, lb, 1e-5)
    close(o["y"], y)
    for a, c in zip(M.mhc_layer_norm_backward_ref(x, lw, mean.float(), rstd.float(), gx),
                    S.layer_norm_bwd(x, lw, mean, rstd, gx)):
        close(a, c)
