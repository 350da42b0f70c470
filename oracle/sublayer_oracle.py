"""The sublayer operators (layer norm, linear layer, gated feed-forward block) in float64,
from their formulas: what the CUDA kernels are tested against.  Any device."""
import math

import torch


def act(name, z):
    """The activation and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))   # 1 + erf would cancel in the negative tail
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    # 0.5 (1 + tanh(u)) = sigmoid(2u), which does not cancel in the negative tail
    c = math.sqrt(2 / math.pi)
    u = 2 * c * (z + 0.044715 * z ** 3)
    p, q = torch.sigmoid(u), torch.sigmoid(-u)
    return z * p, p + z * p * q * 2 * c * (1 + 3 * 0.044715 * z * z)


def layer_norm(x, weight, bias, eps):
    x = x.double()
    mean = x.mean(-1)
    c = x - mean[..., None]
    rstd = 1 / torch.sqrt(c.square().mean(-1) + eps)
    y = c * rstd[..., None]
    if weight is not None:
        y = y * weight.double()
    if bias is not None:
        y = y + bias.double()
    return y, mean, rstd


def layer_norm_bwd(x, weight, mean, rstd, gy):
    x, gy, mean, rstd = x.double(), gy.double(), mean.double()[:, None], rstd.double()[:, None]
    xh = (x - mean) * rstd
    h = gy * weight.double() if weight is not None else gy
    gx = rstd * (h - h.mean(-1, keepdim=True) - xh * (h * xh).mean(-1, keepdim=True))
    return gx, (gy * xh).sum(0), gy.sum(0)


def linear(x, weight, bias, residual, name):
    z = x.double() @ weight.double().t()
    if bias is not None:
        z = z + bias.double()
    y = act(name, z)[0]
    return (y + residual.double() if residual is not None else y), z


def linear_bwd(x, weight, z, gy, name):
    gz = gy.double()
    if name != "none":
        gz = gz * act(name, z.double())[1]
    return gz @ weight.double(), gz.t() @ x.double(), gz.sum(0)


def gated_ffn(x, wg, wu, wd, name):
    gate, up = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    return (act(name, gate)[0] * up) @ wd.double().t(), gate, up


def gated_ffn_bwd(x, wg, wu, wd, gate, up, gy, name):
    x, gy, u = x.double(), gy.double(), up.double()
    a, da = act(name, gate.double())
    gh = gy @ wd.double()
    gg, gu = gh * u * da, gh * a
    return gg @ wg.double() + gu @ wu.double(), gg.t() @ x, gu.t() @ x, gy.t() @ (a * u)
