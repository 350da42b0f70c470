"""The layer norm's rings of rows in shared memory past their first fill: every block has more
rows than stages, so that stages are refilled, phases turn and the slots of the sums alternate.

Rows of up to 2048 elements go to 16 / 2 = 8 blocks an SM at most, up to 4096 to 4, up to 8192 to
2, and a ring has 16 stages at most: with 148 SMs more than 18944, 9472 and 4736 rows."""
import pytest
import torch

import FlagOS_mhc as M
from tests import test_gpu_sublayer as G

pytestmark = pytest.mark.gpu
# widths whose last warp and last pack are full, and others
SHAPES = [(24001, 520), (24001, 1000), (24001, 1024), (20011, 2048), (12001, 2056), (12001, 4096),
          (6001, 4104), (6001, 7168), (5003, 8192)]


def same(a, b):
    return all(p is q or torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dt", G.DTS + [torch.float32])
@pytest.mark.parametrize("T,D", SHAPES)
def test_rings_past_their_first_fill(T, D, dt):
    x, w, b, gy = G.ln_case(T, D, dt, seed=T + 3 * D)
    o = M.mhc_layer_norm(x, w, b, need_backward=True)
    G.ln_check_fwd(o, x, w, b, 1e-5)
    again = M.mhc_layer_norm(x, w, b, need_backward=True)
    assert same(again.values(), o.values())
    g = M.mhc_layer_norm_backward(x, w, o["mean"], o["rstd"], gy)
    G.ln_check_bwd(g, x, w, o["mean"], o["rstd"], gy)
    assert same(M.mhc_layer_norm_backward(x, w, o["mean"], o["rstd"], gy), g)
    only = M.mhc_layer_norm_backward(x, w, o["mean"], o["rstd"], gy, need_param_grads=False)
    assert torch.equal(only[0], g[0])
    # rows inside a wider buffer
    wide = torch.full((T, D + 16), float("nan"), device=G.DEV, dtype=dt)
    wide[:, 8:8 + D] = x
    v = wide[:, 8:8 + D]
    assert same(M.mhc_layer_norm(v, w, b, need_backward=True).values(), o.values())
    assert same(M.mhc_layer_norm_backward(v, w, o["mean"], o["rstd"], gy), g)


@pytest.mark.parametrize("T,D", [(24001, 1024), (12001, 4096), (6001, 7168)])
def test_ring_rows_keep_to_themselves(T, D):
    """NaN and infinity in one row, in rows before and after it in the same block's ring."""
    x, w, b, gy = G.ln_case(T, D, torch.bfloat16, seed=T + D)
    o = M.mhc_layer_norm(x, w, b, need_backward=True)
    g = M.mhc_layer_norm_backward(x, w, o["mean"], o["rstd"], gy)
    bad = torch.tensor([0, 1, T // 2, T - 1], device=G.DEV)
    keep = torch.ones(T, dtype=torch.bool, device=G.DEV)
    keep[bad] = False
    x2, gy2 = x.clone(), gy.clone()
    x2[bad, 17] = torch.tensor([float("nan"), float("inf"), float("-inf"), float("nan")],
                               device=G.DEV).bfloat16()
    gy2[bad, 5] = float("nan")
    o2 = M.mhc_layer_norm(x2, w, b, need_backward=True)
    assert torch.isnan(o2["y"][bad]).all()
    assert all(torch.equal(o2[k][keep], o[k][keep]) for k in o)
    g2 = M.mhc_layer_norm_backward(x2, w, o2["mean"], o2["rstd"], gy2)
    assert torch.isnan(g2[0][bad]).all() and torch.equal(g2[0][keep], g[0][keep])
