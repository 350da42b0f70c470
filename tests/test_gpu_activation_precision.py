"""The activations and their derivatives in fp32, below the rounding of their 16-bit outputs.

Forward: the epilogue adds the residual in fp32, so y = act(z) - r with r the rounded exact value
holds what the rounding of act(z) alone would hide.  Backward: grad_bias sums the unrounded
derivatives of two tokens, of which the second has derivative 1 and grad_y = -r.

Bounds, relative to the terms that are added: __expf(x) is off by 2 + 1.173 |x| units of 2^-23,
the fast division by 2, each rounding by half a unit; the fit of the normal distribution function
by 1.1e-6."""
import math

import pytest
import torch

import FlagOS_mhc as M
from oracle import sublayer_oracle as S
from tests.test_gpu_sublayer import DEV, DTS, tiny_of, u_of

pytestmark = pytest.mark.gpu
U = 2.0 ** -23
C, K = math.sqrt(2 / math.pi), 0.044715


def span(name):
    """Beyond it the exponential leaves fp32's normal range: the functions are 0, or z, there."""
    return {"gelu": 12.0, "gelu_tanh": 8.0, "silu": 80.0, "relu": 80.0}[name]


def points(name, dt):
    a = span(name)
    v = torch.cat([torch.linspace(-a, a, 4001), torch.linspace(-2, 2, 2000), torch.tensor([0.0, 1e-3, -1e-3])])
    return v.to(DEV).to(dt)


def errors(name, z):
    """Error bounds of the value and of the derivative, for z in fp64."""
    if name == "relu":
        return torch.zeros_like(z), torch.zeros_like(z)
    a, da = S.act(name, z)
    if name == "gelu":
        phi = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        e = U * (3 + 1.173 * 0.5 * z * z + 0.5 * z * z)     # of exp(-z^2 / 2), its argument rounded
        # the fit gives the smaller tail; 1 - tail rounds
        d = torch.minimum(cdf, 1 - cdf) * (1.1e-6 + e + 20 * U) + U * cdf
        return z.abs() * d + 2 * U * a.abs(), d + z.abs() * phi * (e + 4 * U) + 2 * U * da.abs()
    arg = z if name == "silu" else 2 * C * z * (1 + K * z * z)
    s = torch.sigmoid(arg)
    n = torch.sigmoid(-arg)
    d = s * (n * U * (2 + 1.173 * arg.abs() + 3 * arg.abs()) + 4 * U)
    slope = 1 if name == "silu" else 2 * C * (1 + 3 * K * z * z)
    # s (1 + z (1 - s) slope): 1 - s is off by d and by a rounding of s
    return z.abs() * d + 2 * U * a.abs(), \
        d + (z * slope).abs() * (d * (n + s) + s * (n * 4 * U + U * s)) + 4 * U * da.abs()


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("few", [True, False])
def test_values(name, dt, few):
    z = points(name, dt)
    if few:
        z = z[:8 * (z.numel() // 8)].reshape(8, -1)      # 8 tokens: z in the features
        x = torch.eye(8, device=DEV, dtype=dt)
        w = z.t().contiguous()
    else:
        z = z[:, None]
        x, w = z, torch.ones(1, 1, device=DEV, dtype=dt)
    a = S.act(name, z.double())[0]
    r = a.to(dt)
    got = M.mhc_linear(x, w, residual=-r, activation=name)["y"].double()
    want = a - r.double()
    e = errors(name, z.double())[0]
    over = (got - want).abs() - (u_of(dt) * (want.abs() + e) + e + tiny_of(dt) + 2.0 ** -126)
    assert over.max() <= 0, (over.max().item(), z.reshape(-1)[over.argmax()].item())


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
def test_derivatives(name, dt):
    z = points(name, dt)
    F = z.numel()
    zz = torch.stack([z, torch.full_like(z, 100.0)])
    da = S.act(name, z.double())[1]
    r = da.to(dt)
    gy = torch.stack([torch.ones_like(z), -r])
    x = torch.zeros(2, 8, device=DEV, dtype=dt)
    w = torch.zeros(F, 8, device=DEV, dtype=dt)
    got = M.mhc_linear_backward(x, w, zz, gy, activation=name, need_x_grad=False,
                                need_weight_grad=False)[2].double()
    want = da - r.double()
    e = errors(name, z.double())[1] + U * r.double().abs()
    over = (got - want).abs() - (u_of(dt) * (want.abs() + e) + e + tiny_of(dt) + 2.0 ** -126)
    assert over.max() <= 0, (over.max().item(), z.reshape(-1)[over.argmax()].item())
