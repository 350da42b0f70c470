"""The sublayer entry points' argument handling, on machines without a GPU: a call that passes
its checks stops at the device check there, so that null and made-up pointers are never read."""
import ctypes
import itertools

import pytest
import torch

from FlagOS_mhc import _C

pytestmark = pytest.mark.skipif(torch.cuda.is_available(),
                                reason="calls with made-up pointers must not reach a GPU")
P = 1 << 20          # an aligned address
WS = ctypes.c_void_p(1 << 21)


def off(ld, p=P):
    """Whether a matrix at p with rows ld apart is unaligned; one that is not there is not."""
    return p is not None and bool((p | ld * 2) & 15)


# rows padded to 16 bytes around odd widths, rows that are not, and even widths
SIZES = [(T, D, F, pad) for T in (4, 64, 200, 1300) for D, F in ((1001, 64), (64, 71), (129, 255), (136, 264))
         for pad in (0, 1)]


def ld(n, pad):
    return (n + 7) // 8 * 8 if pad else n


def passes(status):
    assert status not in (_C.MHC_ERR_WORKSPACE, _C.MHC_ERR_INVALID_ARGUMENT), status


@pytest.mark.parametrize("T,D,F,pad", SIZES)
def test_linear_forward_takes_the_queried_workspace(T, D, F, pad):
    L = _C.lib()
    # the stride of a residual that is not there does not count, whatever it is
    for res, rs in ((None, 0), (None, F), (None, 7), (P, ld(F, pad)), (P, F + 1)):
        un = off(ld(D, pad)) or off(F) or (res is not None and off(rs))
        n = L.mhc_linear_fwd_workspace_bytes(T, D, F, 2, int(un))
        passes(L.mhc_linear_fwd(P, ld(D, pad), P, ld(D, pad), None, res, rs, T, D, F, 2, 4, P, P,
                                WS, n, None))


@pytest.mark.parametrize("act", [0, 4])
@pytest.mark.parametrize("T,D,F,pad", SIZES)
def test_linear_backward_takes_the_queried_workspace(T, D, F, pad, act):
    L = _C.lib()
    for gx, gw, gb in itertools.product((None, P), repeat=3):
        un = off(ld(D, pad)) or off(ld(F, pad)) or off(D, gx) or off(D, gw)
        n = L.mhc_linear_bwd_workspace_bytes(T, D, F, 2, act, int(un))
        passes(L.mhc_linear_bwd(P, ld(D, pad), P, ld(D, pad), P if act else None, ld(F, pad), P,
                                ld(F, pad), T, D, F, 2, act, gx, gw, gb, WS, n, None))


@pytest.mark.parametrize("T,D,F,pad", SIZES)
def test_gated_ffn_takes_the_queried_workspace(T, D, F, pad):
    L = _C.lib()
    d, f = ld(D, pad), ld(F, pad)
    n = L.mhc_gated_ffn_fwd_workspace_bytes(T, D, F, 2, int(off(d) or off(f) or off(D)))
    for gu in (None, P):
        passes(L.mhc_gated_ffn_fwd(P, d, P, d, P, d, P, f, T, D, F, 2, 4, P, gu, gu, f, WS, n, None))
    for gx, gg, gu, gd in itertools.product((None, P), repeat=4):
        un = off(d) or off(f) or off(D, gx) or off(D, gg) or off(D, gu) or off(F, gd)
        n = L.mhc_gated_ffn_bwd_workspace_bytes(T, D, F, 2, int(un))
        passes(L.mhc_gated_ffn_bwd(P, d, P, d, P, d, P, f, P, P, f, P, d, T, D, F, 2, 4, gx, gg, gu,
                                   gd, WS, n, None))


def test_gate_and_up_in_fp32_are_a_flag_on_the_dtype():
    L, f32 = _C.lib(), _C.MHC_GATE_UP_F32
    for dt in (1, 2):
        n = L.mhc_gated_ffn_fwd_workspace_bytes(40, 136, 264, dt | f32, 0)
        assert n == L.mhc_gated_ffn_fwd_workspace_bytes(40, 136, 264, dt, 0) > 0
        passes(L.mhc_gated_ffn_fwd(P, 136, P, 136, P, 136, P, 264, 40, 136, 264, dt | f32, 4, P, P, P, 264,
                                   WS, n, None))
        n = L.mhc_gated_ffn_bwd_workspace_bytes(40, 136, 264, dt | f32, 0)
        assert n == L.mhc_gated_ffn_bwd_workspace_bytes(40, 136, 264, dt, 0) > 0
        passes(L.mhc_gated_ffn_bwd(P, 136, P, 136, P, 136, P, 264, P, P, 264, P, 136, 40, 136, 264, dt | f32,
                                   4, P, P, P, P, WS, n, None))
    # the operands stay 16 bits, and no other operator takes the flag
    assert L.mhc_gated_ffn_fwd(P, 16, P, 16, P, 16, P, 8, 4, 16, 8, f32, 4, P, P, P, 8, WS, 1 << 20,
                               None) == _C.MHC_ERR_UNSUPPORTED_DTYPE
    assert L.mhc_linear_fwd(P, 16, P, 16, None, None, 0, 4, 16, 8, 2 | f32, 4, P, None, None, 0,
                            None) == _C.MHC_ERR_UNSUPPORTED_DTYPE


def test_a_backward_without_outputs_has_nothing_to_do():
    """No device, no workspace: the calls return before either is asked for."""
    L = _C.lib()
    for act, z in ((0, None), (4, P)):
        for T in (0, 4, 200):
            assert L.mhc_linear_bwd(P, 16, P, 16, z, 8, P, 8, T, 16, 8, 2, act, None, None, None, None,
                                    0, None) == _C.MHC_OK
    for T in (0, 4, 200):
        assert L.mhc_gated_ffn_bwd(P, 16, P, 16, P, 16, P, 8, P, P, 8, P, 16, T, 16, 8, 2, 4, None,
                                   None, None, None, None, 0, None) == _C.MHC_OK
    # the arguments are checked all the same
    assert L.mhc_linear_bwd(P, 16, P, 16, None, 8, P, 8, 4, 16, 8, 2, 4, None, None, None, None, 0,
                            None) == _C.MHC_ERR_INVALID_ARGUMENT
    assert L.mhc_gated_ffn_bwd(P, 16, P, 16, P, 16, P, 8, P, None, 8, P, 16, 4, 16, 8, 2, 4, None, None,
                               None, None, None, 0, None) == _C.MHC_ERR_INVALID_ARGUMENT
