"""The autograd wrappers of the sublayer operators, on the CPU: the operators they call are
replaced by their pure-PyTorch definitions."""
import pytest
import torch

import FlagOS_mhc as M
from FlagOS_mhc import autograd as A


@pytest.fixture
def kept(monkeypatch):
    """What each forward was asked to keep."""
    seen = []

    def linear(x, weight, bias=None, residual=None, activation="none", need_backward=False):
        seen.append(need_backward)
        return M.mhc_linear_ref(x, weight, bias, residual, activation)

    def gated(x, w_gate, w_up, w_down, activation="silu", need_backward=False,
              kept_dtype=torch.float32):
        seen.append(need_backward)
        return M.mhc_gated_ffn_ref(x, w_gate, w_up, w_down, activation)

    def linear_bwd(x, weight, z, grad_y, activation="none", need_x_grad=True, need_weight_grad=True,
                   need_bias_grad=True):
        g = M.mhc_linear_backward_ref(x, weight, z, grad_y, activation)
        return tuple(v if n else None for v, n in zip(g, (need_x_grad, need_weight_grad, need_bias_grad)))

    def gated_bwd(*a, activation="silu", need_grads=(True,) * 4):
        g = M.mhc_gated_ffn_backward_ref(*a, activation=activation)
        return tuple(v if n else None for v, n in zip(g, need_grads))

    monkeypatch.setattr(A, "mhc_linear", linear)
    monkeypatch.setattr(A, "mhc_gated_ffn", gated)
    monkeypatch.setattr(A, "mhc_linear_backward", linear_bwd)
    monkeypatch.setattr(A, "mhc_gated_ffn_backward", gated_bwd)
    return seen


def leaves(*shapes, grad):
    g = torch.Generator().manual_seed(1)
    return [torch.randn(*s, generator=g).requires_grad_(k) for s, k in zip(shapes, grad)]


LIN = [(5, 8), (6, 8), (6,), (5, 6)]
FFN = [(5, 8), (6, 8), (6, 8), (8, 6)]


def test_nothing_is_kept_for_a_backward_that_cannot_come(kept):
    lin, ffn = leaves(*LIN, grad=[True] * 4), leaves(*FFN, grad=[True] * 4)
    with torch.no_grad():
        y = M.mhc_linear_fn(*lin, activation="silu")
        f = M.mhc_gated_ffn_fn(*ffn)
    assert kept == [False, False] and not y.requires_grad and not f.requires_grad
    with torch.inference_mode():
        M.mhc_linear_fn(*lin, activation="silu")
        M.mhc_gated_ffn_fn(*ffn)
    M.mhc_linear_fn(*leaves(*LIN, grad=[False] * 4), activation="silu")
    M.mhc_gated_ffn_fn(*leaves(*FFN, grad=[False] * 4))
    M.mhc_linear_fn(*leaves(*LIN[:2], grad=[False] * 2))
    assert not any(kept) and len(kept) == 7


@pytest.mark.parametrize("i", range(4))
def test_one_leaf_is_enough(kept, i):
    one = [k == i for k in range(4)]
    lin, ffn = leaves(*LIN, grad=one), leaves(*FFN, grad=one)
    M.mhc_linear_fn(*lin, activation="silu").sum().backward()
    M.mhc_gated_ffn_fn(*ffn).sum().backward()
    assert kept == [True, True]
    for t in (lin, ffn):
        assert [v.grad is not None for v in t] == one
        assert t[i].grad.shape == t[i].shape


def test_the_functions_keep_by_default(kept):
    lin, ffn = leaves(*LIN, grad=[True] * 4), leaves(*FFN, grad=[True] * 4)
    M.MhcLinearFn.apply(*lin, "gelu").sum().backward()
    M.MhcGatedFfnFn.apply(*ffn, "silu").sum().backward()
    assert kept == [True, True] and all(t.grad is not None for t in lin + ffn)
