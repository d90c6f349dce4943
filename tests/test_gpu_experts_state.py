"""MXExperts keeps its packed weights in its state: saved and loaded, the layer is the same bit for bit."""
import io

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
E, K, H, F, T = 4, 2, 64, 96, 12


def layer(seed, fmt, inner=F):
    from mxq import nn
    g = torch.Generator().manual_seed(seed)
    return nn.MXExperts(torch.randn(E, 2 * inner, H, generator=g).to(DEV) / 8, torch.randn(E, H, inner, generator=g).to(DEV) / 8, fmt)


def inputs():
    from mxq import nn
    g = torch.Generator().manual_seed(5)
    x = torch.randn(T, H, generator=g).to(DEV)
    return (x, *nn.route(torch.randn(T, E, generator=g).to(DEV), K))


@pytest.mark.parametrize("fmt", ["MXFP8_E4M3", "MXFP8_E5M2", "MXFP6_E3M2", "MXFP4"])
def test_saved_and_loaded(fmt):
    a, b = layer(1, fmt), layer(2, fmt)
    state = io.BytesIO()
    torch.save(a.state_dict(), state)
    assert {"up_codes", "up_scales", "down_codes", "down_scales"} <= set(a.state_dict())
    assert all(isinstance(t, torch.Tensor) for t in a.state_dict().values())
    want = a(*inputs())
    assert not torch.equal(b(*inputs()), want)
    state.seek(0)
    b.load_state_dict(torch.load(state, weights_only=True))
    assert torch.equal(b(*inputs()), want)
    whole = torch.nn.Sequential(torch.nn.Linear(H, E), layer(3, fmt)).to(DEV)
    whole.load_state_dict({**whole.state_dict(), **{f"1.{n}": t for n, t in a.state_dict().items()}})
    assert torch.equal(whole[1](*inputs()), want)


def test_the_format_comes_with_the_weights():
    """Codes of another 8-bit format have the same shape: they are read as what they are."""
    a, b = layer(1, "MXFP8_E5M2"), layer(2, "MXFP8_E4M3")
    b.load_state_dict(a.state_dict())
    assert (b.up_fmt, b.down_fmt) == ("MXFP8_E5M2", "MXFP8_E5M2") and torch.equal(b(*inputs()), a(*inputs()))


def test_loading_nothing_is_an_error():
    with pytest.raises(RuntimeError, match="up_codes"):
        layer(1, "MXFP8_E4M3").load_state_dict({})
    with pytest.raises(RuntimeError, match="size mismatch"):
        layer(1, "MXFP8_E4M3").load_state_dict(layer(1, "MXFP8_E4M3", inner=128).state_dict())
