"""The sublayer operators on the GPU against the float64 oracle.

Tolerances count roundings.  u = finfo(dtype).eps / 2 is the largest relative error of one
rounding.  A product of K terms accumulated in fp32, in any order, is off by at most
(K + 64) 2^-24 sum|a||b|.  Where a rounded intermediate (h, gg, gu, gz) enters a product,
u sum|a||b| is added, and u |out| for the output's own rounding.  These bounds are worst
cases; next to them the 2-norm of the error is held to one u per rounding stage (the
roundings of one stage are independent, each u / sqrt(3) at most in the mean square)."""
import pytest
import torch

import FlagOS_mhc as M
from oracle import sublayer_oracle as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTS = [torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def u_of(dt):
    return torch.finfo(dt).eps / 2


def tiny_of(dt):
    """Half a step among the subnormals: the absolute error of a rounding near zero."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def gam(K):
    return (K + 64) * 2.0 ** -24


def rnd(*shape, seed, dt, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dt)


def check(got, want, bound, what, stages=None):
    """|got - want| <= bound elementwise; with stages, the 2-norm within stages * u too."""
    g = got.double()
    assert torch.isfinite(g).all(), what
    err = (g - want).abs()
    over = (err - bound).max().item()
    assert over <= 0, (what, over, err.max().item())
    if stages is not None and want.numel() >= 64:
        rel = (err.norm() / want.norm().clamp_min(1e-300)).item()
        assert rel <= stages * u_of(got.dtype) + 1e-5, (what, rel)


# ------------------------------------------------------------------ layer norm
LN_SHAPES = [(1, 1), (3, 2), (1, 4096), (5, 7), (33, 64), (130, 1001), (257, 768), (7, 7168),
             (1000, 1024), (19, 8192), (4, 20000), (2000, 40), (3, 12289)]


def ln_slack(D):
    # depth of any sum over a row: D/32 serial additions and a tree, at 2^-24 each
    return (D / 32 + 24) * 2.0 ** -24


def ln_case(T, D, dt, seed, affine=True):
    x = rnd(T, D, seed=seed, dt=torch.float32) * (1 + torch.arange(T, device=DEV)[:, None] % 3)
    x = (x + rnd(T, 1, seed=seed + 1, dt=torch.float32)).to(dt)
    w = rnd(D, seed=seed + 2, dt=torch.float32) if affine else None
    b = rnd(D, seed=seed + 3, dt=torch.float32) if affine else None
    return x, w, b, rnd(T, D, seed=seed + 4, dt=dt)


def ln_check_fwd(o, x, w, b, eps):
    T, D = x.shape
    y, mean, rstd = S.layer_norm(x, w, b, eps)
    e, xd = ln_slack(D), x.double()
    dmean = e * xd.abs().mean(1)
    # the variance is the mean of (x - mean)^2: off by e, and by (dmean)^2
    var = (xd - mean[:, None]).square().mean(1) + eps
    drel = e + dmean.square() / var
    check(o["mean"], mean, dmean + 2.0 ** -24 * mean.abs(), "mean")
    check(o["rstd"], rstd, (drel + 2.0 ** -22) * rstd, "rstd")
    xh = (xd - mean[:, None]) * rstd[:, None]
    wa = w.double().abs() if w is not None else 1.0
    ba = b.double().abs() if b is not None else 0.0
    slack = wa * ((dmean * rstd)[:, None] + xh.abs() * (drel + 2.0 ** -21)[:, None]
                  + 2.0 ** -23 * (xd.abs() + mean.abs()[:, None]) * rstd[:, None])
    check(o["y"], y, u_of(x.dtype) * (y.abs() + slack) + slack + 2.0 ** -23 * (y.abs() + ba)
          + tiny_of(x.dtype), "y", None if x.dtype == torch.float32 else 1)


@pytest.mark.parametrize("dt", DTS + [torch.float32])
@pytest.mark.parametrize("T,D", LN_SHAPES)
def test_layer_norm_forward(T, D, dt):
    x, w, b, _ = ln_case(T, D, dt, seed=T + D)
    ln_check_fwd(M.mhc_layer_norm(x, w, b, eps=1e-5, need_backward=True), x, w, b, 1e-5)
    o = M.mhc_layer_norm(x, eps=1e-3)
    assert set(o) == {"y"}
    o = M.mhc_layer_norm(x, eps=1e-3, need_backward=True)
    ln_check_fwd(o, x, None, None, 1e-3)


def ln_check_bwd(got, x, w, mean, rstd, gy):
    T, D = x.shape
    gx, gw, gb = S.layer_norm_bwd(x, w, mean, rstd, gy)
    e = ln_slack(D) + 2.0 ** -20
    xd, m, r = x.double(), mean.double()[:, None], rstd.double()[:, None]
    # x - mean is one rounding of the difference; xh two more
    xh = ((xd - m) * r).abs()
    h = gy.double().abs() * (w.double().abs() if w is not None else 1.0)
    s1, s2 = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
    slack = e * r * (h + s1 + xh * s2)
    check(got[0], gx, u_of(x.dtype) * (gx.abs() + slack) + slack + tiny_of(x.dtype), "gx",
          None if x.dtype == torch.float32 else 1.5)
    if got[1] is not None:
        # any order of T additions
        et = (T + 64) * 2.0 ** -24
        check(got[1], gw, et * (gy.double().abs() * xh).sum(0) + 1e-30, "gw")
        check(got[2], gb, et * gy.double().abs().sum(0) + 1e-30, "gb")


@pytest.mark.parametrize("dt", DTS + [torch.float32])
@pytest.mark.parametrize("T,D", LN_SHAPES)
def test_layer_norm_backward(T, D, dt):
    x, w, b, gy = ln_case(T, D, dt, seed=2 * T + D)
    o = M.mhc_layer_norm(x, w, b, need_backward=True)
    ln_check_bwd(M.mhc_layer_norm_backward(x, w, o["mean"], o["rstd"], gy), x, w, o["mean"],
                 o["rstd"], gy)
    got = M.mhc_layer_norm_backward(x, None, o["mean"], o["rstd"], gy, need_param_grads=False)
    assert got[1] is None and got[2] is None
    ln_check_bwd(got, x, None, o["mean"], o["rstd"], gy)


def test_layer_norm_views_types_and_repeats():
    x, w, b, gy = ln_case(70, 264, torch.bfloat16, seed=9)
    want = M.mhc_layer_norm(x, w, b, need_backward=True)
    wide = rnd(70, 300, seed=1, dt=torch.bfloat16)
    for off in (0, 3, 8):          # rows that start anywhere
        wide[:, off:off + 264] = x
        v = wide[:, off:off + 264]
        o = M.mhc_layer_norm(v, w, b, need_backward=True)
        g = M.mhc_layer_norm_backward(v, w, o["mean"], o["rstd"], gy)
        ref = M.mhc_layer_norm_backward(x, w, want["mean"], want["rstd"], gy)
        ln_check_fwd(o, x, w, b, 1e-5)
        ln_check_bwd(g, x, w, o["mean"], o["rstd"], gy)
        # rows 600 bytes apart are read element by element: a thread sums other elements
        # than with 16-byte packs, so the sums may differ by their bounds, checked above
    buf = torch.zeros(70, 304, device=DEV, dtype=torch.bfloat16)
    for off in (0, 8):             # packs as in the packed tensor: the same sums
        buf[:, off:off + 264] = x
        v = buf[:, off:off + 264]
        o = M.mhc_layer_norm(v, w, b, need_backward=True)
        g = M.mhc_layer_norm_backward(v, w, o["mean"], o["rstd"], gy)
        assert torch.equal(o["y"], want["y"])
        assert all(torch.equal(p, q) for p, q in zip(g, ref))
    x3 = x.reshape(2, 35, 264)
    assert torch.equal(M.mhc_layer_norm(x3, w, b)["y"], want["y"].reshape(2, 35, 264))
    xt = x.t().contiguous().t()    # columns contiguous: packed first
    assert torch.equal(M.mhc_layer_norm(xt, w, b)["y"], want["y"])
    wb = M.mhc_layer_norm(x, w.bfloat16(), b.bfloat16())["y"]
    assert torch.equal(wb, M.mhc_layer_norm(x, w.bfloat16().float(), b.bfloat16().float())["y"])
    a = M.mhc_layer_norm_backward(x, w, want["mean"], want["rstd"], gy)
    c = M.mhc_layer_norm_backward(x, w, want["mean"], want["rstd"], gy)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    # a broadcast grad_y (stride 0)
    one = torch.ones(1, 1, device=DEV, dtype=torch.bfloat16).expand(70, 264)
    ln_check_bwd(M.mhc_layer_norm_backward(x, w, want["mean"], want["rstd"], one), x, w,
                 want["mean"], want["rstd"], one)


def test_layer_norm_special_rows():
    x, w, b, gy = ln_case(6, 512, torch.bfloat16, seed=4)
    clean = M.mhc_layer_norm(x, w, b, need_backward=True)
    bad = x.clone()
    bad[2, 17] = float("nan")
    bad[3, 5] = float("inf")
    bad[4] = 3.0                   # constant row: zero variance
    o = M.mhc_layer_norm(bad, w, b, need_backward=True)
    assert torch.isnan(o["y"][2]).all() and torch.isnan(o["y"][3]).all()
    assert torch.equal(o["y"][4], b.bfloat16())
    for i in (0, 1, 5):
        assert torch.equal(o["y"][i], clean["y"][i])
    big = torch.full((2, 256), 3e38, device=DEV, dtype=torch.float32)
    assert M.mhc_layer_norm(big)["y"].shape == big.shape     # overflows to inf - inf, no fault
    off = (rnd(4, 4096, seed=5, dt=torch.float32) + 1000.0)  # a mean far from zero
    ln_check_fwd(M.mhc_layer_norm(off, eps=1e-5, need_backward=True), off, None, None, 1e-5)


# ------------------------------------------------------------------ linear
LIN_SHAPES = [(1, 1, 1), (1, 8, 8), (2, 5, 7), (3, 64, 200), (17, 72, 40), (9, 520, 1000),
              (33, 1000, 264), (64, 256, 512), (65, 129, 255), (130, 264, 136), (257, 328, 513),
              (300, 1024, 640), (513, 2048, 256), (1, 4096, 1032), (8, 3000, 2048),
              (48, 1536, 768), (1100, 257, 515), (2100, 1030, 771)]


def lin_case(T, D, F, dt, seed):
    return (rnd(T, D, seed=seed, dt=dt), rnd(F, D, seed=seed + 1, dt=dt, scale=D ** -0.5),
            rnd(F, seed=seed + 2, dt=dt), rnd(T, F, seed=seed + 3, dt=dt),
            rnd(T, F, seed=seed + 4, dt=dt))


def act_slack(z):
    """Of the fast exponential and division: the activation's value and derivative."""
    return 1e-5 * (1 + z.abs())


def lin_check_fwd(o, x, w, b, r, name):
    dt, u = x.dtype, u_of(x.dtype)
    y, z = S.linear(x, w, b, r, name)
    mag = x.double().abs() @ w.double().abs().t()
    dz = gam(x.shape[-1]) * mag + 2.0 ** -22 * z.abs()
    # |act'| <= 1.13 for each of the activations
    dy = 1.2 * dz + (act_slack(z) * S.act(name, z)[0].abs() + 1e-7 if name != "none" else 0)
    check(o["y"], y, dy + u * (y.abs() + dy) + 2.0 ** -23 * y.abs() + tiny_of(dt), "y", 1)
    if o.get("z") is not None:
        check(o["z"], z, dz + u * (z.abs() + dz) + tiny_of(dt), "z", 1)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("T,D,F", LIN_SHAPES)
def test_linear_forward(T, D, F, dt):
    x, w, b, r, _ = lin_case(T, D, F, dt, seed=T + D + F)
    for name in ACTS:
        o = M.mhc_linear(x, w, bias=b, residual=r, activation=name, need_backward=True)
        assert (o["z"] is None) == (name == "none")
        lin_check_fwd(o, x, w, b, r, name)
        y = M.mhc_linear(x, w, bias=b, residual=r, activation=name)["y"]
        assert torch.equal(y, o["y"])
    lin_check_fwd(M.mhc_linear(x, w), x, w, None, None, "none")
    lin_check_fwd(M.mhc_linear(x, w, residual=r), x, w, None, r, "none")


def lin_check_bwd(got, x, w, z, gy, name):
    dt, u = x.dtype, u_of(x.dtype)
    T, (F, D) = x.shape[0], w.shape
    want = S.linear_bwd(x, w, z, gy, name)
    gz = gy.double()
    dgz = torch.zeros_like(gz)
    if name != "none":
        da = S.act(name, z.double())[1]
        dgz = gz.abs() * act_slack(z.double())
        gz = gz * da
    dgz_r = dgz + (u * gz.abs() + tiny_of(dt) if name != "none" else 0)  # rounded operand
    ga, stages = gz.abs() + dgz_r, 1 if name == "none" else 2
    wa, xa = w.double().abs(), x.double().abs()
    if got[0] is not None:
        b = gam(F) * (ga @ wa) + dgz_r @ wa
        check(got[0], want[0], b + u * (want[0].abs() + b) + tiny_of(dt), "gx", stages)
    if got[1] is not None:
        b = gam(T) * (ga.t() @ xa) + dgz_r.t() @ xa
        check(got[1], want[1], b + u * (want[1].abs() + b) + tiny_of(dt), "gw", stages)
    if got[2] is not None:
        b = gam(T) * ga.sum(0) + dgz.sum(0)
        check(got[2], want[2], b + u * (want[2].abs() + b) + tiny_of(dt), "gb", 1.5)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("T,D,F", LIN_SHAPES)
def test_linear_backward(T, D, F, dt):
    x, w, b, r, gy = lin_case(T, D, F, dt, seed=T + 2 * D + F)
    for name in ACTS:
        z = M.mhc_linear(x, w, bias=b, activation=name, need_backward=True)["z"]
        lin_check_bwd(M.mhc_linear_backward(x, w, z, gy, activation=name), x, w, z, gy, name)


def test_linear_backward_only_what_is_needed():
    x, w, b, r, gy = lin_case(40, 136, 72, torch.bfloat16, seed=3)
    z = M.mhc_linear(x, w, activation="silu", need_backward=True)["z"]
    full = M.mhc_linear_backward(x, w, z, gy, activation="silu")
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 0, 0)):
        got = M.mhc_linear_backward(x, w, z, gy, activation="silu", need_x_grad=bool(need[0]),
                                    need_weight_grad=bool(need[1]), need_bias_grad=bool(need[2]))
        for n, p, q in zip(need, got, full):
            assert (p is None) if not n else torch.equal(p, q)


@pytest.mark.parametrize("T", [5, 200])
@pytest.mark.parametrize("D,F", [(136, 264), (100, 60)])
def test_linear_views(T, D, F):
    dt = torch.bfloat16
    x, w, b, r, gy = lin_case(T, D, F, dt, seed=T + D)
    want = M.mhc_linear(x, w, bias=b, residual=r, activation="gelu", need_backward=True)
    gwant = M.mhc_linear_backward(x, w, want["z"], gy, activation="gelu")
    for off in (0, 8, 3):
        def wide(t):
            buf = torch.full((t.shape[0], t.shape[1] + 24), float("nan"), device=DEV, dtype=dt)
            buf[:, off:off + t.shape[1]] = t
            return buf[:, off:off + t.shape[1]]
        o = M.mhc_linear(wide(x), wide(w), bias=b, residual=wide(r), activation="gelu",
                         need_backward=True)
        assert torch.equal(o["y"], want["y"]) and torch.equal(o["z"], want["z"])
        g = M.mhc_linear_backward(wide(x), wide(w), wide(want["z"]), wide(gy), activation="gelu")
        assert all(torch.equal(p, q) for p, q in zip(g, gwant))
    wt = w.t().contiguous().t()
    assert torch.equal(M.mhc_linear(x, wt, bias=b, residual=r, activation="gelu")["y"], want["y"])
    # one row for all tokens
    rb = r[:1].expand(T, F)
    lin_check_fwd(M.mhc_linear(x, w, residual=rb), x, w, None, rb, "none")
    ge = gy[:, :1].expand(T, F)
    lin_check_bwd(M.mhc_linear_backward(x, w, None, ge), x, w, None, ge, "none")


def test_activations_over_their_range():
    """One column of weight 1 makes z the input itself."""
    for dt in DTS:
        v = torch.cat([torch.linspace(-30, 30, 2001), torch.tensor([0.0, -0.0, 1e-30, 6e4, -6e4])])
        x = v.to(DEV).to(dt)[:, None]
        one, gy = torch.ones(1, 1, device=DEV, dtype=dt), torch.ones(v.numel(), 1, device=DEV, dtype=dt)
        for name in ACTS:
            a, da = S.act(name, x.double())
            y = M.mhc_linear(x, one, activation=name)["y"]
            tol = (u_of(dt) + act_slack(x.double())) * a.abs() + 1e-7
            check(y, a, tol, name)
            gx = M.mhc_linear_backward(x, one, x, gy, activation=name)[0]
            check(gx, da, 2 * u_of(dt) * da.abs() + act_slack(x.double().clamp(-12, 12)), name + "'")


@pytest.mark.parametrize("T", [3, 40, 600])
def test_activations_beyond_the_type(T):
    """A pre-activation past fp16's range: the forward works in fp32, z is kept as infinity, and
    the derivative there is 0 or 1."""
    dt = torch.float16
    x = torch.full((T, 8), 250.0, device=DEV, dtype=dt)
    w = torch.zeros(16, 8, device=DEV, dtype=dt)
    w[0], w[1] = 250.0, -250.0            # z = 5e5, -5e5
    gy = torch.ones(T, 16, device=DEV, dtype=dt)
    for name in ("relu", "gelu", "gelu_tanh", "silu"):
        o = M.mhc_linear(x, w, activation=name, need_backward=True)
        assert torch.isinf(o["z"][:, :2]).all() and (o["y"][:, 1:] == 0).all()
        gx, gw, gb = M.mhc_linear_backward(x, w, o["z"], gy, activation=name)
        assert torch.isfinite(gx).all() and (gx[:, 0] == 250.0).all(), name
        assert gb[0] == T and gb[1] == 0
    up = torch.ones_like(w)
    f = M.mhc_gated_ffn(x / 250, w * 400, up / 8, w.t().contiguous() * 0 + 1, need_backward=True)
    g = M.mhc_gated_ffn_backward(x / 250, w * 0, up / 8, w.t().contiguous() * 0 + 1,
                                 torch.full_like(f["gate"], float("-inf")), f["up"], x / 250)
    assert all(torch.isfinite(t).all() for t in g)


def test_rows_keep_to_themselves():
    """NaN and infinity in one token reach that token's outputs only."""
    for T in (6, 200):
        x, w, b, r, _ = lin_case(T, 136, 264, torch.bfloat16, seed=T)
        want = M.mhc_linear(x, w, bias=b, activation="silu")["y"]
        x2 = x.clone()
        x2[3, 7], x2[4, 1] = float("nan"), float("inf")
        got = M.mhc_linear(x2, w, bias=b, activation="silu")["y"]
        keep = torch.ones(T, dtype=torch.bool, device=DEV)
        keep[3] = keep[4] = False
        assert torch.equal(got[keep], want[keep]) and torch.isnan(got[3]).all()


# ------------------------------------------------------------------ gated feed-forward
FFN_SHAPES = [(1, 1, 1), (1, 64, 72), (2, 7, 5), (5, 200, 136), (16, 512, 1000), (33, 264, 520),
              (64, 1024, 512), (65, 100, 255), (140, 328, 264), (257, 136, 1023), (300, 512, 384),
              (3, 4096, 640), (48, 768, 2048), (1100, 257, 131), (1300, 520, 1290)]


def ffn_case(T, D, F, dt, seed):
    return (rnd(T, D, seed=seed, dt=dt), rnd(F, D, seed=seed + 1, dt=dt, scale=D ** -0.5),
            rnd(F, D, seed=seed + 2, dt=dt, scale=D ** -0.5),
            rnd(D, F, seed=seed + 3, dt=dt, scale=F ** -0.5), rnd(T, D, seed=seed + 4, dt=dt))


def ffn_check_fwd(o, x, wg, wu, wd, name):
    dt, u = x.dtype, u_of(x.dtype)
    D, F = x.shape[-1], wg.shape[0]
    y, gate, up = S.gated_ffn(x, wg, wu, wd, name)
    xa = x.double().abs()
    dg, du = gam(D) * (xa @ wg.double().abs().t()), gam(D) * (xa @ wu.double().abs().t())
    if "gate" in o:
        check(o["gate"], gate, dg + u * (gate.abs() + dg) + tiny_of(dt), "gate", 1)
        check(o["up"], up, du + u * (up.abs() + du) + tiny_of(dt), "up", 1)
    a = S.act(name, gate)[0].abs()
    da = 1.2 * dg + act_slack(gate) * a + 1e-7
    dh = da * (up.abs() + du) + a * du
    dh = dh + u * (a * up.abs() + dh) + tiny_of(dt)
    wa = wd.double().abs().t()
    b = dh @ wa + gam(F) * ((a * up.abs() + dh) @ wa)
    check(o["y"], y, b + u * (y.abs() + b) + tiny_of(dt), "y", 2)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("T,D,F", FFN_SHAPES)
def test_gated_ffn_forward(T, D, F, dt):
    x, wg, wu, wd, _ = ffn_case(T, D, F, dt, seed=T + D + F)
    for name in ACTS:
        o = M.mhc_gated_ffn(x, wg, wu, wd, activation=name, need_backward=True)
        ffn_check_fwd(o, x, wg, wu, wd, name)
        assert torch.equal(M.mhc_gated_ffn(x, wg, wu, wd, activation=name)["y"], o["y"])


def ffn_check_bwd(got, x, wg, wu, wd, gate, up, gy, name):
    dt, u = x.dtype, u_of(x.dtype)
    T, D, F = x.shape[0], x.shape[1], wg.shape[0]
    want = S.gated_ffn_bwd(x, wg, wu, wd, gate, up, gy, name)
    xa, gya = x.double().abs(), gy.double().abs()
    a, da = S.act(name, gate.double())
    ua = up.double().abs()
    gh = (gy.double() @ wd.double()).abs()
    dgh = gam(D) * (gya @ wd.double().abs())
    sl = act_slack(gate.double())

    def operand(v, dv):  # value, its error with the rounding to dtype
        return v + dv, dv + u * (v + dv) + tiny_of(dt)

    gg, dgg = operand(gh * ua * da.abs(), dgh * ua * (da.abs() + sl) + gh * ua * sl)
    gu, dgu = operand(gh * a.abs(), dgh * (a.abs() * (1 + sl) + 1e-7) + gh * (a.abs() * sl + 1e-7))
    h, dh = operand(a.abs() * ua, (a.abs() * sl + 1e-7) * ua)
    wga, wua = wg.double().abs(), wu.double().abs()
    bounds = [dgg @ wga + dgu @ wua + gam(2 * F) * (gg @ wga + gu @ wua),
              dgg.t() @ xa + gam(T) * (gg.t() @ xa), dgu.t() @ xa + gam(T) * (gu.t() @ xa),
              gya.t() @ dh + gam(T) * (gya.t() @ h)]
    for g, w, b, what in zip(got, want, bounds, ("gx", "gwg", "gwu", "gwd")):
        if g is not None:
            check(g, w, 1.01 * b + u * (w.abs() + b) + tiny_of(dt), what, 2)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("T,D,F", FFN_SHAPES)
def test_gated_ffn_backward(T, D, F, dt):
    x, wg, wu, wd, gy = ffn_case(T, D, F, dt, seed=T + D + 3 * F)
    for name in ACTS:
        o = M.mhc_gated_ffn(x, wg, wu, wd, activation=name, need_backward=True)
        got = M.mhc_gated_ffn_backward(x, wg, wu, wd, o["gate"], o["up"], gy, activation=name)
        ffn_check_bwd(got, x, wg, wu, wd, o["gate"], o["up"], gy, name)
    again = M.mhc_gated_ffn_backward(x, wg, wu, wd, o["gate"], o["up"], gy, activation=name)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("T", [4, 150])
def test_gated_ffn_views_and_needs(T):
    x, wg, wu, wd, gy = ffn_case(T, 136, 264, torch.bfloat16, seed=T)
    o = M.mhc_gated_ffn(x, wg, wu, wd, need_backward=True)
    full = M.mhc_gated_ffn_backward(x, wg, wu, wd, o["gate"], o["up"], gy)
    both = torch.cat([wg, wu])     # halves of one weight
    g2, u2 = both.chunk(2)
    wide = torch.full((T, 200), float("nan"), device=DEV, dtype=x.dtype)
    wide[:, 5:141] = x
    o2 = M.mhc_gated_ffn(wide[:, 5:141], g2, u2, wd, need_backward=True)
    assert torch.equal(o2["y"], o["y"]) and torch.equal(o2["gate"], o["gate"])
    inter = torch.stack([o["gate"], o["up"]], 1)     # gate and up interleaved by rows
    got = M.mhc_gated_ffn_backward(wide[:, 5:141], g2, u2, wd, inter[:, 0], inter[:, 1], gy)
    assert all(torch.equal(p, q) for p, q in zip(got, full))
    for need in ((1, 0, 0, 0), (0, 1, 0, 1), (0, 0, 1, 0), (0, 0, 0, 0)):
        got = M.mhc_gated_ffn_backward(x, wg, wu, wd, o["gate"], o["up"], gy,
                                       need_grads=[bool(n) for n in need])
        for n, p, q in zip(need, got, full):
            assert (p is None) if not n else torch.equal(p, q)
    same = M.mhc_gated_ffn(x, wg, wg, wd, need_backward=True)     # one weight for both
    ffn_check_fwd(same, x, wg, wg, wd, "silu")
    assert torch.equal(same["gate"], same["up"])


# ------------------------------------------------------------------ empty batches, streams, graphs
def test_no_tokens():
    x, wg, wu, wd, gy = ffn_case(0, 64, 72, torch.bfloat16, seed=1)
    o = M.mhc_gated_ffn(x, wg, wu, wd, need_backward=True)
    assert o["y"].shape == (0, 64) and o["gate"].shape == (0, 72)
    g = M.mhc_gated_ffn_backward(x, wg, wu, wd, o["gate"], o["up"], gy)
    assert g[0].shape == (0, 64) and all((t == 0).all() for t in g[1:])
    o = M.mhc_linear(x, wg, activation="silu", need_backward=True)
    g = M.mhc_linear_backward(x, wg, o["z"], o["y"], activation="silu")
    assert g[0].shape == (0, 64) and (g[1] == 0).all() and (g[2] == 0).all()
    w = torch.ones(64, device=DEV)
    o = M.mhc_layer_norm(x, w, w, need_backward=True)
    g = M.mhc_layer_norm_backward(x, w, o["mean"], o["rstd"], gy)
    assert g[0].shape == (0, 64) and (g[1] == 0).all() and (g[2] == 0).all()


def sub_step(d):
    o = M.mhc_layer_norm(d["x"], d["lw"], d["lb"], need_backward=True)
    f = M.mhc_gated_ffn(o["y"], d["wg"], d["wu"], d["wd"], need_backward=True)
    p = M.mhc_linear(f["y"], d["w"], bias=d["b"], residual=d["x"], activation="gelu",
                     need_backward=True)
    gp = M.mhc_linear_backward(f["y"], d["w"], p["z"], d["gy"], activation="gelu")
    gf = M.mhc_gated_ffn_backward(o["y"], d["wg"], d["wu"], d["wd"], f["gate"], f["up"], gp[0])
    gn = M.mhc_layer_norm_backward(d["x"], d["lw"], o["mean"], o["rstd"], gf[0])
    return [o["y"], f["y"], p["y"], *gp, *gf, *gn]


def sub_inputs(T, D, F, dt, seed):
    x, wg, wu, wd, gy = ffn_case(T, D, F, dt, seed)
    return dict(x=x, wg=wg, wu=wu, wd=wd, gy=gy, w=rnd(D, D, seed=seed + 9, dt=dt, scale=D ** -0.5),
                b=rnd(D, seed=seed + 10, dt=dt), lw=rnd(D, seed=seed + 11, dt=torch.float32),
                lb=rnd(D, seed=seed + 12, dt=torch.float32))


SUB = [(3, 264, 520), (40, 100, 60), (300, 256, 512), (1100, 512, 1032)]


@pytest.mark.parametrize("T,D,F", SUB)
def test_graph_replay_matches_eager(T, D, F):
    d = sub_inputs(T, D, F, torch.bfloat16, seed=T)
    sub_step(d)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            outs = sub_step(d)
    torch.cuda.synchronize()
    for rep in range(2):
        new = sub_inputs(T, D, F, torch.bfloat16, seed=100 + rep)
        for k, v in new.items():
            d[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(outs, sub_step(new))):
            assert torch.equal(a, b), (rep, i)
    from FlagOS_mhc import _C
    assert _C.lib().mhc_device_status() == 0


@pytest.mark.parametrize("T", [5, 300])
def test_captured_training_step(T):
    """Forward and backward through the autograd wrappers, captured once and replayed on new
    inputs, against the eager step (made after the graph's own leaves are done with)."""
    D, F = 136, 264

    def leaves(d):
        return {k: d[k].clone().requires_grad_() for k in ("x", "lw", "lb", "wg", "wu", "wd", "w", "b")}

    def step(q, gy):
        h = M.mhc_gated_ffn_fn(M.mhc_layer_norm_fn(q["x"], q["lw"], q["lb"]), q["wg"], q["wu"], q["wd"])
        y = M.mhc_linear_fn(h, q["w"], q["b"], residual=q["x"], activation="gelu")
        return [y.detach(), *torch.autograd.grad(y, list(q.values()), gy)]

    d = sub_inputs(T, D, F, torch.bfloat16, seed=3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        q = leaves(d)
        step(q, d["gy"])                   # warm-up on the capturing stream
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        outs = step(q, d["gy"])
    for seed in (21, 22):
        new = sub_inputs(T, D, F, torch.bfloat16, seed=seed)
        with torch.no_grad():
            for k in q:
                q[k].copy_(new[k])
        d["gy"].copy_(new["gy"])
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(outs, step(leaves(new), new["gy"]))):
            assert torch.equal(a, b), (seed, i)


@pytest.mark.parametrize("T,D,F", SUB)
def test_two_streams_at_once(T, D, F):
    ds = [sub_inputs(T, D, F, torch.bfloat16, seed=7 + i) for i in range(2)]
    want = [sub_step(d) for d in ds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ds]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = sub_step(ds[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_offsets_past_32_bits():
    """Outputs of more than 2^31 elements: the last rows are right too."""
    T, D, F = 140000, 16, 16384
    x, w, b, r, _ = lin_case(8, D, F, torch.bfloat16, seed=5)
    xl = torch.zeros(T, D, device=DEV, dtype=torch.bfloat16)
    xl[-8:] = x
    y = M.mhc_linear(xl, w, bias=b, activation="relu")["y"]
    lin_check_fwd({"y": y[-8:]}, x, w, b, None, "relu")
    assert torch.equal(y[0], torch.relu(b))
    del y
    xn = torch.zeros(T, F, device=DEV, dtype=torch.bfloat16)
    xn[-3:] = rnd(3, F, seed=6, dt=torch.bfloat16)
    o = M.mhc_layer_norm(xn, need_backward=True)
    ln_check_fwd({k: v[-3:] for k, v in o.items()}, xn[-3:], None, None, 1e-5)
    g = M.mhc_layer_norm_backward(xn, None, o["mean"], o["rstd"], xn)
    del o
    assert torch.isfinite(g[0][-3:]).all() and (g[0][0] == 0).all()


# ------------------------------------------------------------------ a layer, with autograd
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("B,S_,N,D,F", [(2, 33, 4, 128, 328), (1, 3, 4, 256, 512), (2, 150, 8, 64, 200)])
def test_layer_with_autograd(B, S_, N, D, F, dt):
    """pre -> norm -> gated block -> linear -> post, against float64 automatic
    differentiation.  The chain rounds to dtype at y, norm, h, block, linear and out going
    forward and as often going back: 16 u in the 2-norm covers each twice over the small
    factors of the norm and the streams' mixing."""
    g = torch.Generator().manual_seed(1)
    hm = N * (N + 2)

    def leaf(*shape, scale=1.0, to=dt):
        return (torch.randn(*shape, generator=g) * scale).to(to).to(DEV).requires_grad_()

    p = dict(x=leaf(B, S_, N, D), phi=leaf(hm, N * D, scale=(N * D) ** -0.5, to=torch.float32),
             alpha=leaf(3, to=torch.float32), base=leaf(hm, scale=0.1, to=torch.float32),
             lw=leaf(D, to=torch.float32), lb=leaf(D, to=torch.float32),
             wg=leaf(F, D, scale=D ** -0.5), wu=leaf(F, D, scale=D ** -0.5),
             wd=leaf(D, F, scale=F ** -0.5), w=leaf(D, D, scale=D ** -0.5), b=leaf(D))
    gy = torch.randn(B, S_, N, D, generator=g).to(dt).to(DEV)
    y, post, comb = M.mhc_pre_clamp_sinkhorn_fn(p["x"], p["phi"], p["alpha"], p["base"])
    n = M.mhc_layer_norm_fn(y, p["lw"], p["lb"])
    f = M.mhc_gated_ffn_fn(n, p["wg"], p["wu"], p["wd"])
    h = M.mhc_linear_fn(f, p["w"], p["b"], residual=y, activation="gelu_tanh")
    out = M.mhc_post_fn(p["x"], comb.reshape(B, S_, N, N), h, post.reshape(B, S_, N))
    out.backward(gy)

    q = {k: v.detach().double().cpu().requires_grad_() for k, v in p.items()}
    xf = q["x"].reshape(-1, N, D)
    flat = xf.reshape(-1, N * D)
    mix = (flat * (flat.square().mean(1, keepdim=True) + 1e-6).rsqrt()) @ q["phi"].t()
    al, ba = q["alpha"], q["base"]
    o = {"post_out": 2 * torch.sigmoid(mix[:, N:2 * N] * al[1] + ba[N:2 * N]),
         "y": (xf * (torch.sigmoid(mix[:, :N] * al[0] + ba[:N]) + 1e-6)[:, :, None]).sum(1)}
    m = torch.softmax((mix[:, 2 * N:] * al[2] + ba[2 * N:]).reshape(-1, N, N), -1) + 1e-6
    m = m / (m.sum(1, keepdim=True) + 1e-6)
    for _ in range(19):
        m = m / (m.sum(2, keepdim=True) + 1e-6)
        m = m / (m.sum(1, keepdim=True) + 1e-6)
    o["comb_frag"] = m
    yn, _, _ = S.layer_norm(o["y"], q["lw"], q["lb"], 1e-5)
    fy, _, _ = S.gated_ffn(yn, q["wg"], q["wu"], q["wd"], "silu")
    hy, _ = S.linear(fy, q["w"], q["b"], o["y"], "gelu_tanh")
    want = torch.einsum("tji,tjd->tid", o["comb_frag"], xf) + \
        o["post_out"][:, :, None] * hy[:, None, :]
    want.backward(gy.double().cpu().reshape(want.shape))
    tol = 16 * u_of(dt)
    e = (out.detach().double().cpu().reshape(want.shape) - want).norm() / want.norm()
    assert e <= tol, ("out", e.item())
    for k in p:
        a, b = p[k].grad.double().cpu(), q[k].grad
        e = ((a - b).norm() / b.norm()).item()
        ok = p[k].grad.dtype == p[k].dtype and e <= tol
        assert ok, (k, e)


def test_gradients_against_differences():
    """Directional derivatives of a scalar of each operator against central differences of
    the float64 oracle, at the same point."""
    dt = torch.float16
    x, wg, wu, wd, gy = ffn_case(12, 40, 56, dt, seed=2)
    lw = rnd(40, seed=20, dt=torch.float32)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    M.mhc_gated_ffn_fn(*leaves).backward(gy)
    for i, t in enumerate(leaves):
        d = rnd(*t.shape, seed=30 + i, dt=torch.float64)
        args = [v.detach().double() for v in leaves]
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + 1e-4 * d, args[i] - 1e-4 * d
        num = ((S.gated_ffn(*hi, "silu")[0] - S.gated_ffn(*lo, "silu")[0]) * gy.double()).sum() / 2e-4
        got = (t.grad.double() * d).sum()
        # each gradient element is off by a few u of its size, at random
        tol = 6 * u_of(dt) * (t.grad.double().norm() * d.norm()) / t.numel() ** 0.5 * 4 + 1e-4
        assert abs(got - num) <= tol, (i, got.item(), num.item())
    xl, wl = x.clone().requires_grad_(), lw.clone().requires_grad_()
    M.mhc_layer_norm_fn(xl, wl).backward(gy)
    for i, t in enumerate((xl, wl)):
        d = rnd(*t.shape, seed=40 + i, dt=torch.float64)
        args = [xl.detach().double(), wl.detach().double()]
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + 1e-4 * d, args[i] - 1e-4 * d
        num = ((S.layer_norm(*hi, None, 1e-5)[0] - S.layer_norm(*lo, None, 1e-5)[0])
               * gy.double()).sum() / 2e-4
        got = (t.grad.double() * d).sum()
        tol = 6 * u_of(dt) * (t.grad.double().norm() * d.norm()) / t.numel() ** 0.5 * 4 + 1e-4
        assert abs(got - num) <= tol, (i, got.item(), num.item())


def test_first_call_of_a_thread():
    """A thread whose first CUDA work is one of these calls (autograd's backward thread is
    such a thread) has no current context yet."""
    import threading
    x, wg, wu, wd, gy = ffn_case(200, 64, 72, torch.bfloat16, seed=8)
    o = M.mhc_gated_ffn(x, wg, wu, wd, need_backward=True)
    want = M.mhc_gated_ffn_backward(x, wg, wu, wd, o["gate"], o["up"], gy)
    calls = [lambda: [M.mhc_gated_ffn(x, wg, wu, wd)["y"]], lambda: [M.mhc_linear(x, wg)["y"]],
             lambda: M.mhc_gated_ffn_backward(x, wg, wu, wd, o["gate"], o["up"], gy)]
    wants = [[o["y"]], [M.mhc_linear(x, wg)["y"]], want]
    for call, w in zip(calls, wants):
        got = []
        th = threading.Thread(target=lambda: got.append(call()))
        th.start()
        th.join()
        torch.cuda.synchronize()
        assert got and all(torch.equal(p, q) for p, q in zip(got[0], w))


def test_native_kernels_run():
    from FlagOS_mhc import _C
    n0 = _C.lib().mhc_kernel_launches()
    x, wg, wu, wd, gy = ffn_case(4, 64, 64, torch.bfloat16, seed=1)
    M.mhc_gated_ffn(x, wg, wu, wd)
    M.mhc_linear(x, wg)
    M.mhc_layer_norm(x)
    assert _C.lib().mhc_kernel_launches() >= n0 + 4
