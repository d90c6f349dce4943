"""The epilogue's activations relative to their own size over the whole of float32: the packed outputs turn a relative error into
steps of the code, so a tail has to be as exact as the middle. The references are in float64 without cancellation (erfc,
x sigmoid). Bounds: every rounding and the hardware's exp2 (2^-22.5) and reciprocal (2^-23) sum to 14 units of 2^-24 at most;
2^-20, plus the smallest normal float for what passes below it."""
import math

import pytest
import torch

from _feedforward import FORMATS, assert_packed

pytestmark = pytest.mark.gpu
DEV = "cuda"
EXACT = {
    "silu": lambda v: v * torch.sigmoid(v),
    "gelu": lambda v: 0.5 * v * torch.special.erfc(-v * math.sqrt(0.5)),
    "gelu_tanh": lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)),
}


def through(values, activation, rows, out):
    """act(values) as the products give it: the bias carries the argument, the sum adds zero."""
    from mxq import nn
    n = values.numel()
    x = (torch.zeros(rows, 32, dtype=torch.uint8, device=DEV), torch.full((rows, 1), 127, dtype=torch.uint8, device=DEV))
    w = (torch.zeros(n, 32, dtype=torch.uint8, device=DEV), torch.full((n, 1), 127, dtype=torch.uint8, device=DEV))
    return nn.linear_packed(x, w, "MXFP8_E4M3", bias=values.to(DEV), activation=activation, out=out)


def arguments():
    near = torch.linspace(-16, 16, 160001)
    far = torch.linspace(-110, 110, 110001)
    tiny = torch.exp2(torch.linspace(-126, 0, 5000))
    return torch.cat((near, far, tiny, -tiny, torch.tensor([-87.3, -87.34, -87.5, -88.0, -89.0, -90.0, -91.9, -1e3, -1e10, -3e38, 3e38])))


@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("activation", sorted(EXACT))
def test_relative(activation, rows):
    v = arguments()
    got = through(v, activation, rows, torch.float32)[rows - 1].cpu().double()
    want = EXACT[activation](v.double())
    off, tol = (got - want).abs(), 2.0 ** -20 * want.abs() + 2.0 ** -126
    worst = int((off / tol).argmax())
    assert (off <= tol).all(), (float(v[worst]), float(got[worst]), float(want[worst]), float((off / tol).max()))


@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("activation", sorted(EXACT))
def test_packed_in_the_tail(activation, rows):
    """Blocks that lie in the negative tail as a whole: the codes are those of the exact values but for a near tie."""
    for low, high in ((-4.5, -4.0), (-6.0, -5.5), (-8.0, -7.5), (-9.3, -9.0)):
        v = torch.linspace(low, high, 320)
        want = EXACT[activation](v.double()).to(DEV)[None].expand(rows, -1)
        for fmt in sorted(FORMATS):
            assert_packed(through(v, activation, rows, fmt), want, 2.0 ** -20 * want.abs(), fmt, f"{activation} {low} {fmt}")
