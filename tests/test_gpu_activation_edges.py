"""The epilogue's activations at the ends of float32, through products with a single one in K: large and small arguments, both
Infs, NaN, zeros of both signs; and their accuracy in between, against float64 (a few ulp: 2^-21 of the argument and the
result, as float32 evaluations of the same formulas have it)."""
import math

import pytest
import torch

from _feedforward import act64

pytestmark = pytest.mark.gpu
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def through(values, activation, rows):
    """act(values) as the products give it: bias carries the argument, the sum adds zero."""
    from mxq import nn
    n = values.numel()
    x = (torch.zeros(rows, 32, dtype=torch.uint8, device="cuda"), torch.full((rows, 1), 127, dtype=torch.uint8, device="cuda"))
    w = (torch.zeros(n, 32, dtype=torch.uint8, device="cuda"), torch.full((n, 1), 127, dtype=torch.uint8, device="cuda"))
    return nn.linear_packed(x, w, "MXFP8_E4M3", bias=values.cuda(), activation=activation, out=torch.float32)


@pytest.mark.parametrize("rows", [1, 700])
@pytest.mark.parametrize("activation", ACTS)
def test_ends(activation, rows):
    v = torch.tensor([0.0, -0.0, 1e-38, -1e-38, 1e-45, 87.0, -87.0, 89.0, -89.0, 104.0, -104.0, 1e4, -1e4, 3e38, -3e38, math.inf,
                      -math.inf, math.nan])
    y = through(v, activation, rows)
    assert torch.equal(y.nan_to_num(7e7), y[:1].expand_as(y).nan_to_num(7e7))
    y, want = y[0].cpu().double(), act64(v.double(), activation)
    for a, g, t in zip(v.tolist(), y.tolist(), want.tolist()):
        if a == -math.inf and activation not in (None, "relu"):
            assert math.isnan(g), (activation, a, g)         # -Inf * 0
        elif math.isnan(t) or math.isinf(t):
            assert g == t or math.isnan(g) and math.isnan(t), (activation, a, g)
        else:
            assert abs(g - t) <= 2.0 ** -21 * max(abs(t), min(abs(a), 8.0)) + 1e-36, (activation, a, g, t)


@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("activation", ACTS)
def test_accuracy(activation, rows):
    v = torch.cat((torch.linspace(-12, 12, 20001), torch.linspace(-0.01, 0.01, 2001)))
    y = through(v, activation, rows)[rows - 1].cpu().double()
    want = act64(v.double(), activation)
    tol = 2.0 ** -21 * torch.maximum(want.abs(), v.double().abs().clamp_max(8.0)) + 1e-36
    off = (y - want).abs()
    assert (off <= tol).all(), float((off / tol).max())
