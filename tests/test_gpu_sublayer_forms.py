"""Every kernel form of the linear layer's and the gated block's matrix products against the
float64 oracle, at sizes that reach it (``sublayer_forms``, whose lists are checked for
completeness on the CPU).  The bounds are those of ``test_gpu_sublayer``."""
import pytest
import torch

import FlagOS_mhc as M
from FlagOS_mhc import _C
from tests import sublayer_forms as SF
from tests import test_gpu_sublayer as G

pytestmark = pytest.mark.gpu
DTS = [torch.bfloat16, torch.float16]


def same(a, b):
    return all(p is q or torch.equal(p, q) for p, q in zip(a, b))


@pytest.fixture(autouse=True)
def clean():
    yield
    torch.cuda.empty_cache()            # the fp64 intermediates of a test are a few GB
    assert _C.lib().mhc_device_status() == 0


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("i", range(len(SF.LINEAR_SHAPES)), ids=lambda i: "%d-%d-%d" % SF.LINEAR_SHAPES[i])
def test_linear_forms(i, dt):
    T, D, F = SF.LINEAR_SHAPES[i]
    name = G.ACTS[(i + 2 * DTS.index(dt)) % 5]
    x, w, b, r, gy = G.lin_case(T, D, F, dt, seed=1000 + i)
    o = M.mhc_linear(x, w, bias=b, residual=r, activation=name, need_backward=True)
    G.lin_check_fwd(o, x, w, b, r, name)
    assert torch.equal(M.mhc_linear(x, w, bias=b, residual=r, activation=name)["y"], o["y"])
    g = M.mhc_linear_backward(x, w, o["z"], gy, activation=name)
    G.lin_check_bwd(g, x, w, o["z"], gy, name)
    assert same(M.mhc_linear_backward(x, w, o["z"], gy, activation=name), g)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("i", range(len(SF.GATED_SHAPES)), ids=lambda i: "%d-%d-%d" % SF.GATED_SHAPES[i])
def test_gated_forms(i, dt):
    T, D, F = SF.GATED_SHAPES[i]
    name = G.ACTS[(i + 2 * DTS.index(dt)) % 5]
    x, wg, wu, wd, gy = G.ffn_case(T, D, F, dt, seed=2000 + i)
    o = M.mhc_gated_ffn(x, wg, wu, wd, activation=name, need_backward=True)
    G.ffn_check_fwd(o, x, wg, wu, wd, name)
    assert torch.equal(M.mhc_gated_ffn(x, wg, wu, wd, activation=name)["y"], o["y"])
    g = M.mhc_gated_ffn_backward(x, wg, wu, wd, o["gate"], o["up"], gy, activation=name)
    G.ffn_check_bwd(g, x, wg, wu, wd, o["gate"], o["up"], gy, name)
    # the same with gate and up packed: unaligned rows where F is odd
    again = M.mhc_gated_ffn_backward(x, wg, wu, wd, o["gate"].contiguous(), o["up"].contiguous(), gy,
                                     activation=name)
    assert same(again, g)
    # gate and up kept in 16 bits: rounded once, and read back as the same values
    h = M.mhc_gated_ffn(x, wg, wu, wd, activation=name, need_backward=True, kept_dtype=dt)
    assert same(h.values(), [o["y"], o["gate"].to(dt), o["up"].to(dt)])
    g = M.mhc_gated_ffn_backward(x, wg, wu, wd, h["gate"], h["up"], gy, activation=name)
    for gate, up in ((h["gate"].float(), h["up"].float()), (h["gate"].contiguous(), h["up"].contiguous())):
        assert same(M.mhc_gated_ffn_backward(x, wg, wu, wd, gate, up, gy, activation=name), g)
