"""Calls of the sublayer operators that the documentation allows, apart from sizes and values:
outputs that are not wanted, rows inside wider buffers."""
import itertools

import pytest
import torch

import FlagOS_mhc as M

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = torch.bfloat16


def rnd(*shape, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV).to(DT)


def padded(t):
    """The same rows, 16-byte aligned inside a wider buffer of NaN."""
    n = t.shape[1]
    buf = torch.full((t.shape[0], (n + 7) // 8 * 8 + 8), float("nan"), device=DEV, dtype=DT)
    buf[:, :n] = t
    return buf[:, :n]


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("T,D,F", [(6, 1001, 64), (200, 1001, 64), (200, 129, 255), (600, 64, 71)])
def test_any_subset_of_gradients_of_padded_rows(T, D, F, act):
    x, w, wu = rnd(T, D, seed=1), rnd(F, D, seed=2) / 8, rnd(F, D, seed=3) / 8
    wd, gy, gf = rnd(D, F, seed=4) / 8, rnd(T, D, seed=5), rnd(T, F, seed=6)
    z = M.mhc_linear(x, w, activation=act, need_backward=True)["z"]
    full = M.mhc_linear_backward(x, w, z, gf, activation=act)
    zp = padded(z) if z is not None else None
    for need in itertools.product((False, True), repeat=3):
        got = M.mhc_linear_backward(padded(x), padded(w), zp, padded(gf), activation=act,
                                    need_x_grad=need[0], need_weight_grad=need[1],
                                    need_bias_grad=need[2])
        for n, p, q in zip(need, got, full):
            assert torch.equal(p, q) if n else p is None, need
    o = M.mhc_gated_ffn(x, w, wu, wd, activation=act, need_backward=True)
    full = M.mhc_gated_ffn_backward(x, w, wu, wd, o["gate"], o["up"], gy, activation=act)
    for need in itertools.product((False, True), repeat=4):
        got = M.mhc_gated_ffn_backward(padded(x), padded(w), padded(wu), padded(wd), o["gate"],
                                       o["up"], padded(gy), activation=act, need_grads=need)
        for n, p, q in zip(need, got, full):
            assert torch.equal(p, q) if n else p is None, need


def launches():
    from FlagOS_mhc import _C
    return _C.lib().mhc_kernel_launches()


def test_a_backward_without_outputs_launches_nothing():
    T, D, F = 40, 136, 72
    x, w, gy, gf = rnd(T, D, seed=1), rnd(F, D, seed=2), rnd(T, D, seed=3), rnd(T, F, seed=4)
    wd = rnd(D, F, seed=5)
    n = launches()
    assert M.mhc_linear_backward(x, w, gf, gf, activation="silu", need_x_grad=False,
                                 need_weight_grad=False, need_bias_grad=False) == (None,) * 3
    assert M.mhc_gated_ffn_backward(x, w, w, wd, gf, gf, gy, need_grads=(False,) * 4) == (None,) * 4
    assert launches() == n
    some = M.mhc_gated_ffn_backward(x, w, w, wd, gf, gf, gy, need_grads=(i == 2 for i in range(4)))
    assert [t is None for t in some] == [True, True, False, True]
    with pytest.raises(AssertionError):     # the arguments are checked all the same
        M.mhc_linear_backward(x, w, gf, gy, activation="silu", need_x_grad=False,
                              need_weight_grad=False, need_bias_grad=False)


def peak_of(call):
    """Bytes that a call takes at most, its result among them."""
    torch.cuda.synchronize()
    base = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = call()
    return out, torch.cuda.max_memory_allocated() - base


def test_wrappers_without_grad_mode_take_what_the_operator_takes():
    T, D, F = 2048, 256, 4096
    x, w, wu = (t.requires_grad_() for t in (rnd(T, D, seed=1), rnd(F, D, seed=2), rnd(F, D, seed=3)))
    wd = (rnd(D, F, seed=4) / 64).requires_grad_()
    for fn, op in ((lambda: M.mhc_linear_fn(x, w, activation="silu"),
                    lambda: M.mhc_linear(x, w, activation="silu")["y"]),
                   (lambda: M.mhc_gated_ffn_fn(x, w, wu, wd),
                    lambda: M.mhc_gated_ffn(x, w, wu, wd)["y"])):
        with torch.no_grad():
            want, least = peak_of(op)
            got, peak = peak_of(fn)
        assert torch.equal(got, want) and not got.requires_grad and peak == least
        kept, more = peak_of(fn)
        assert torch.equal(kept, want) and kept.requires_grad and more >= least + T * F * 2


def test_a_hosts_own_context_stays_current():
    """A host that made its context with the driver API finds it current after a call; the pointers
    and streams that it hands over belong to it.  The call is one without device work."""
    import ctypes
    import threading
    from FlagOS_mhc import _C
    cu = ctypes.CDLL("libcuda.so.1")
    torch.zeros(1, device=DEV)              # the driver is initialised
    seen = {}

    def host():
        mine, now = ctypes.c_void_p(), ctypes.c_void_p()
        seen["made"] = cu.cuCtxCreate_v2(ctypes.byref(mine), 0, torch.cuda.current_device())
        if seen["made"]:
            return
        p = ctypes.c_void_p(1 << 20)
        seen["status"] = _C.lib().mhc_gated_ffn_bwd(p, 16, p, 16, p, 16, p, 8, p, p, 8, p, 16, 0, 16, 8,
                                                    2, 4, p, None, None, None, None, 0, None)
        cu.cuCtxGetCurrent(ctypes.byref(now))
        seen["kept"] = now.value == mine.value
        cu.cuCtxDestroy_v2(mine)

    th = threading.Thread(target=host)
    th.start()
    th.join()
    assert seen == {"made": 0, "status": 0, "kept": True}


@pytest.mark.parametrize("T", [1, 40, 3000])
def test_sums_over_tokens_with_infinite_terms(T):
    """One infinite gradient makes the sums of its column infinite, two of both signs NaN."""
    D = F = 72
    inf = float("inf")
    x, w, gy = rnd(T, D, seed=1), rnd(F, D, seed=2), rnd(T, F, seed=3)
    at = sorted({0, T // 2, T - 1})
    for k, t in enumerate(at):
        gy[t, k] = inf
        gy[t, 8 + k] = -inf
    gy[at[0], 20], gy[at[-1], 20] = inf, -inf
    gb = M.mhc_linear_backward(x, w, None, gy, need_x_grad=False, need_weight_grad=False)[2]
    want = gy.double().sum(0)
    o = M.mhc_layer_norm(x, need_backward=True)
    gw, gbn = M.mhc_layer_norm_backward(x, None, o["mean"], o["rstd"], gy)[1:]
    xh = (x.double() - o["mean"].double()[:, None]) * o["rstd"].double()[:, None]
    wantw = (gy.double() * xh).sum(0)
    for got, ref in ((gb, want), (gbn, want), (gw, wantw)):
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(torch.isinf(got), torch.isinf(ref))
        odd = torch.isinf(ref)
        assert torch.equal(got[odd].double(), ref[odd])
