"""What the gated block keeps from the forward to the backward, and what its rounding costs."""
import pytest
import torch

import FlagOS_mhc as M
from oracle import sublayer_oracle as S
from tests import test_gpu_sublayer as G

pytestmark = pytest.mark.gpu


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("dt", G.DTS)
@pytest.mark.parametrize("T,D,F", [(4, 512, 1032), (40, 1024, 2048), (600, 512, 1000), (2300, 1032, 2056)])
def test_gradients_against_exact_ones(T, D, F, dt):
    """Against the gradients of the exact forward.  Roundings are independent and each makes the
    2-norm's error of one rounding, e: that of the output and that of the operand h, gg or gu give
    sqrt(2) e with gate and up in fp32.  Kept in 16 bits they add about one e each in the squares,
    the gate's times (g a'(g) / a(g))^2, 1.3 for silu over normal values: sqrt(4.3) e."""
    x, wg, wu, wd, gy = G.ffn_case(T, D, F, dt, seed=T + F)
    gate, up = S.gated_ffn(x, wg, wu, wd, "silu")[1:]
    want = S.gated_ffn_bwd(x, wg, wu, wd, gate, up, gy, "silu")
    for kept, times in ((torch.float32, 1.5), (dt, 2.3)):
        o = M.mhc_gated_ffn(x, wg, wu, wd, need_backward=True, kept_dtype=kept)
        assert o["gate"].dtype == o["up"].dtype == kept
        got = M.mhc_gated_ffn_backward(x, wg, wu, wd, o["gate"], o["up"], gy)
        for a, b, what in zip(got, want, ("gx", "gwg", "gwu", "gwd")):
            e = rel(b.to(dt), b)            # one rounding
            assert rel(a, b) <= times * e + 1e-5, (what, kept, rel(a, b) / e)


def test_autograd_keeps_what_it_is_asked_to():
    dt = torch.bfloat16
    x, wg, wu, wd, gy = G.ffn_case(70, 136, 264, dt, seed=5)
    for kept in (torch.float32, dt):
        leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
        M.mhc_gated_ffn_fn(*leaves, kept_dtype=kept).backward(gy)
        o = M.mhc_gated_ffn(x, wg, wu, wd, need_backward=True, kept_dtype=kept)
        want = M.mhc_gated_ffn_backward(x, wg, wu, wd, o["gate"], o["up"], gy)
        assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))


def test_refusals():
    dt = torch.bfloat16
    x, wg, wu, wd, gy = G.ffn_case(9, 64, 72, dt, seed=6)
    o = M.mhc_gated_ffn(x, wg, wu, wd, need_backward=True)
    for kept in (torch.float16, torch.float64):
        with pytest.raises(ValueError, match="gate and up"):
            M.mhc_gated_ffn(x, wg, wu, wd, need_backward=True, kept_dtype=kept)
        with pytest.raises(ValueError, match="gate and up"):
            M.mhc_gated_ffn_backward(x, wg, wu, wd, o["gate"].to(kept), o["up"].to(kept), gy)
    with pytest.raises(ValueError, match="dtypes"):
        M.mhc_gated_ffn_backward(x, wg, wu, wd, o["gate"], o["up"].to(dt), gy)


@pytest.mark.parametrize("T,F", [(5, 264), (40, 264), (40, 61), (600, 264), (600, 261), (2300, 2060)])
def test_gate_and_up_anywhere(T, F):
    """fp32 rows that start on 4, 16 or 32 bytes, packed or not."""
    dt, D = torch.bfloat16, 136
    x, wg, wu, wd, gy = G.ffn_case(T, D, F, dt, seed=7)
    o = M.mhc_gated_ffn(x, wg, wu, wd, need_backward=True)
    want = M.mhc_gated_ffn_backward(x, wg, wu, wd, o["gate"], o["up"], gy)
    for pad, off in ((0, 0), (8, 0), (4, 4), (7, 1), (12, 3)):
        w = [torch.full((T, F + pad), float("nan"), device=G.DEV) for _ in range(2)]
        for b, k in zip(w, ("gate", "up")):
            b[:, off:off + F] = o[k]
        got = M.mhc_gated_ffn_backward(x, wg, wu, wd, *(b[:, off:off + F] for b in w), gy)
        assert all(torch.equal(p, q) for p, q in zip(got, want)), (pad, off)
    both = torch.stack([o["gate"], o["up"]], 1)
    got = M.mhc_gated_ffn_backward(x, wg, wu, wd, both[:, 0], both[:, 1], gy)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
