"""Cases of the sublayer operators: layer norm, linear layer and gated feed-forward block.

A hyper-connection layer is ``pre -> norm -> sublayer -> post``.  The cases below are the
middle part, at this repository's widths (4096, 7168) and at generic ones.  With ``own``
false, ``run`` computes them in plain fp32 torch operations; with ``own`` true it calls the
FlagOS_mhc entry points.
"""
import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _norm(way, T, D, dtype, sliced=False):
    return {"op": "norm", "way": way, "T": T, "D": D, "dtype": dtype, "sliced": sliced}


def _linear(way, T, D, F, dtype, act, bias, residual, sliced=False):
    return {"op": "linear", "way": way, "T": T, "D": D, "F": F, "dtype": dtype, "act": act,
            "bias": bias, "residual": residual, "sliced": sliced}


def _ffn(way, T, D, F, dtype, act, sliced=False):
    return {"op": "ffn", "way": way, "T": T, "D": D, "F": F, "dtype": dtype, "act": act,
            "sliced": sliced}


def listed():
    named = {
        # one token of a decode step: launch latency
        "norm_fwd_token": _norm("fwd", 1, 4096, "bf16"),
        # a ragged batch at a width that no vector divides, rows inside a wider buffer
        "norm_bwd_odd": _norm("bwd", 1999, 1001, "fp16", True),
        # a training step's tokens at the widest configuration
        "norm_bwd_train": _norm("bwd", 32768, 7168, "bf16"),
        # full-precision activations
        "norm_fwd_fp32": _norm("fwd", 16384, 4096, "fp32"),
        # the sublayer of one token, everything in the epilogue
        "linear_fwd_token": _linear("fwd", 1, 4096, 4096, "bf16", "gelu", True, True),
        # ragged training batch, fp16, sizes that no tile divides
        "linear_train_ragged": _linear("train", 1023, 1000, 2504, "fp16", "gelu_tanh", True, False),
        # the sublayer h_out = y W^T of the eight-stream configuration, forward and backward
        "linear_train_layer": _linear("train", 65536, 4096, 4096, "bf16", "none", False, False),
        # decode: one token, then a batch of tokens; the weights are the traffic
        "ffn_fwd_token": _ffn("fwd", 1, 4096, 16384, "bf16", "silu"),
        "ffn_fwd_batch48": _ffn("fwd", 48, 7168, 14336, "bf16", "silu"),
        # a small training batch of odd length, x inside a wider buffer
        "ffn_train_small": _ffn("train", 509, 2048, 5464, "fp16", "gelu_tanh", True),
        # a prompt
        "ffn_fwd_prompt": _ffn("fwd", 4096, 7168, 14336, "bf16", "silu"),
        # a training step's tokens
        "ffn_train": _ffn("train", 8192, 4096, 16384, "bf16", "silu"),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly whole 16-byte packs, as models have; one in five any size."""
    w = _log(rng, lo, hi)
    return w if rng.random() < 0.2 else max(8, w // 8 * 8)


def draw(rng):
    op = rng.choice(["norm", "linear", "ffn"])
    sliced = rng.random() < 0.25
    if op == "norm":
        D = _width(rng, 64, 8192)
        T = _log(rng, 1, min(65536, 2 ** 28 // D))
        return _norm(rng.choice(["fwd", "bwd"]), T, D, rng.choice(["bf16", "fp16", "fp32"]), sliced)
    way = rng.choice(["fwd", "fwd", "train"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    D, F = _width(rng, 256, 8192), _width(rng, 256, 16384)
    a_token = (2 if op == "linear" else 6) * D * F * (3 if way == "train" else 1)
    T = _log(rng, 1, max(2, min(65536, int(5e12 / a_token))))
    if op == "linear":
        return _linear(way, T, D, F, dtype, rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]),
                       rng.random() < 0.5, rng.random() < 0.5, sliced)
    return _ffn(way, T, D, F, dtype, rng.choice(["silu", "gelu", "gelu_tanh", "relu"]), sliced)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, T, D = _DT[case["dtype"]], case["T"], case["D"]

    def rand(*shape, scale=1.0, to=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(to)

    s = dict(case)
    if case["sliced"]:  # the first D columns of rows that are 64 elements longer
        s["x"] = rand(T, D + 64)[:, :D]
    else:
        s["x"] = rand(T, D)
    if case["op"] == "norm":
        # rows with an offset and a scale of their own, as residual streams have
        s["x"].mul_(torch.rand(T, 1, generator=g, device="cuda") + 0.5)
        s["x"].add_(rand(T, 1, to=torch.float32))
        s["weight"] = rand(D, scale=0.1, to=torch.float32) + 1
        s["bias"] = rand(D, scale=0.1, to=torch.float32)
        if case["way"] == "bwd":
            s["grad_y"] = rand(T, D)
            xf = s["x"].double()
            mean = xf.mean(1)
            s["mean"] = mean.float()
            s["rstd"] = (1 / ((xf - mean[:, None]).square().mean(1) + 1e-5).sqrt()).float()
        return s
    F = case["F"]
    if case["op"] == "linear":
        s["weight"] = rand(F, D, scale=D ** -0.5)
        s["b"] = rand(F, scale=0.5) if case["bias"] else None
        s["res"] = rand(T, F) if case["residual"] else None
        if case["way"] == "train":
            s["grad_y"] = rand(T, F)
        return s
    s["w_gate"] = rand(F, D, scale=D ** -0.5)
    s["w_up"] = rand(F, D, scale=D ** -0.5)
    s["w_down"] = rand(D, F, scale=F ** -0.5)
    if case["way"] == "train":
        s["grad_y"] = rand(T, D)
    return s


# ------------------------------------------------------------------ plain form
def _act(name, z):
    """The activation and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * 2 ** -0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    c = (2 / math.pi) ** 0.5
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return (0.5 * z * (1 + t),
            0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z))


def _plain_norm(s):
    dt, x, w = s["x"].dtype, s["x"].float(), s["weight"]
    if s["way"] == "fwd":
        mean = x.mean(1)
        c = x - mean[:, None]
        rstd = 1 / (c.square().mean(1) + 1e-5).sqrt()
        return [(c * rstd[:, None] * w + s["bias"]).to(dt), mean, rstd]
    gy = s["grad_y"].float()
    xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
    h = gy * w
    gx = s["rstd"][:, None] * (h - h.mean(1, keepdim=True) - xhat * (h * xhat).mean(1, keepdim=True))
    return [gx.to(dt), (gy * xhat).sum(0), gy.sum(0)]


def _plain_linear(s):
    dt, x, w = s["x"].dtype, s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    a, da = _act(s["act"], z)
    y = a if s["res"] is None else a + s["res"].float()
    if s["way"] == "fwd":
        return [y.to(dt)]
    gz = s["grad_y"].float() * da
    out = [y.to(dt), (gz @ w).to(dt), (gz.t() @ x).to(dt)]
    return out + ([gz.sum(0).to(dt)] if s["b"] is not None else [])


def _plain_ffn(s):
    dt, x = s["x"].dtype, s["x"].float()
    wg, wu, wd = s["w_gate"].float(), s["w_up"].float(), s["w_down"].float()
    u = x @ wu.t()
    a, da = _act(s["act"], x @ wg.t())
    h = a * u
    y = (h @ wd.t()).to(dt)
    if s["way"] == "fwd":
        return [y]
    gy = s["grad_y"].float()
    gh = gy @ wd
    gg, gu = gh * u * da, gh * a
    return [y, (gg @ wg + gu @ wu).to(dt), (gg.t() @ x).to(dt), (gu.t() @ x).to(dt),
            (gy.t() @ h).to(dt)]


# ------------------------------------------------------------------ the framework's operators
def _own(s):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    if os.path.join(root, "flagos-mhc_b200") not in sys.path:
        sys.path.insert(0, os.path.join(root, "flagos-mhc_b200"))
    import FlagOS_mhc as M
    train = s["way"] == "train"
    if s["op"] == "norm":
        if s["way"] == "fwd":
            o = M.mhc_layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5, need_backward=True)
            return [o["y"], o["mean"], o["rstd"]]
        return list(M.mhc_layer_norm_backward(s["x"], s["weight"], s["mean"], s["rstd"], s["grad_y"]))
    if s["op"] == "linear":
        o = M.mhc_linear(s["x"], s["weight"], bias=s["b"], residual=s["res"], activation=s["act"],
                         need_backward=train)
        if not train:
            return [o["y"]]
        gx, gw, gb = M.mhc_linear_backward(s["x"], s["weight"], o["z"], s["grad_y"],
                                           activation=s["act"], need_bias_grad=s["b"] is not None)
        return [o["y"], gx, gw] + ([gb] if gb is not None else [])
    o = M.mhc_gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], activation=s["act"],
                        need_backward=train)
    if not train:
        return [o["y"]]
    return [o["y"], *M.mhc_gated_ffn_backward(s["x"], s["w_gate"], s["w_up"], s["w_down"], o["gate"],
                                              o["up"], s["grad_y"], activation=s["act"])]


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "linear": _plain_linear, "ffn": _plain_ffn}[state["op"]](state)


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    T, D = case["T"], case["D"]
    if case["op"] == "norm":
        if case["way"] == "fwd":  # x; y; mean, rstd; weight, bias
            return {"bytes": 2 * T * D * e + 8 * T + 8 * D, "flops": 8 * T * D}
        return {"bytes": 3 * T * D * e + 8 * T + 12 * D, "flops": 16 * T * D}
    F = case["F"]
    train = case["way"] == "train"
    if case["op"] == "linear":
        n = T * D + D * F + T * F * (2 if case["residual"] else 1)
        n += T * F + T * D + D * F if train else 0  # grad_y; grad_x, grad_weight
        n += F * (2 if train else 1) if case["bias"] else 0
        return {"bytes": n * e, "flops": 2 * T * D * F * (3 if train else 1)}
    n = 2 * T * D + 3 * D * F
    n += 2 * T * D + 3 * D * F if train else 0
    return {"bytes": n * e, "flops": 6 * T * D * F * (3 if train else 1)}


# ------------------------------------------------------------------ 64 bits, by automatic differentiation
def exact(case, seed):
    s = prepare(case, seed)
    leaf = {k: v.double().requires_grad_(case["way"] != "fwd") for k, v in s.items()
            if torch.is_tensor(v) and k not in ("grad_y", "mean", "rstd")}

    def act(z):
        if case["act"] == "gelu":  # z times the normal distribution function
            return z * torch.special.ndtr(z)
        if case["act"] == "gelu_tanh":
            return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * z * (1 + 0.044715 * z ** 2))
        return {"none": lambda v: v, "relu": lambda v: torch.clamp(v, min=0),
                "silu": lambda v: v * torch.sigmoid(v)}[case["act"]](z)

    if case["op"] == "norm":
        var, mean = torch.var_mean(leaf["x"], dim=1, correction=0)
        rstd = (var + 1e-5) ** -0.5
        y = torch.addcmul(leaf["bias"], (leaf["x"] - mean[:, None]) * rstd[:, None], leaf["weight"])
        outs, wrt = [y, mean, rstd], ["x", "weight", "bias"]
    elif case["op"] == "linear":
        z = torch.einsum("td,fd->tf", leaf["x"], leaf["weight"])
        y = act(z + leaf["b"] if case["bias"] else z)
        outs = [y + leaf["res"] if case["residual"] else y]
        wrt = ["x", "weight"] + (["b"] if case["bias"] else [])
    else:
        h = act(torch.einsum("td,fd->tf", leaf["x"], leaf["w_gate"])) * \
            torch.einsum("td,fd->tf", leaf["x"], leaf["w_up"])
        outs = [torch.einsum("tf,df->td", h, leaf["w_down"])]
        wrt = ["x", "w_gate", "w_up", "w_down"]
    if case["way"] == "fwd":
        return outs
    grads = list(torch.autograd.grad(outs[0], [leaf[k] for k in wrt], s["grad_y"].double()))
    return grads if case["way"] == "bwd" else [outs[0].detach()] + grads
