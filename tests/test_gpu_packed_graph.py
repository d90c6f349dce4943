"""The products inside an autograd graph: the residual's gradient is the result's, a gradient that would have to pass through x
or a bias raises and is not lost in silence, forward-mode tangents raise, and what asks for no gradient is as it was."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from _feedforward import random_pair

pytestmark = pytest.mark.gpu
DEV = "cuda"


def operands(seed=1, M=5, N=64, K=96):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(M, K, generator=g).to(DEV), random_pair((N, K), "MXFP8_E4M3", g, DEV), torch.randn(N, generator=g).to(DEV),
            torch.randn(M, N, generator=g).to(DEV, torch.bfloat16))


@pytest.mark.parametrize("lead", [(5,), (1, 5)])
@pytest.mark.parametrize("pair", [False, True])
def test_the_residual_has_its_gradient(lead, pair):
    from mxq import block, nn
    x, w, bias, r = operands()
    arg = block.ocp.quantize_packed(x, "MXFP8_E4M3", axis=-1) if pair else x
    shape = lambda t: tuple(v.view(*lead, -1) for v in t) if isinstance(t, tuple) else t.view(*lead, -1)  # noqa: E731
    leaf = r.view(*lead, -1).clone().requires_grad_(True)
    y = nn.linear_packed(shape(arg), w, "MXFP8_E4M3", bias=bias, activation="silu", residual=leaf)
    assert y.requires_grad
    assert torch.equal(y.detach(), nn.linear_packed(shape(arg), w, "MXFP8_E4M3", bias=bias, activation="silu", residual=leaf.detach()))
    dy = torch.randn_like(y)
    y.backward(dy)
    assert torch.equal(leaf.grad, dy)
    part = torch.zeros(5, 70, device=DEV, dtype=torch.bfloat16, requires_grad=True)         # a view of a wider leaf
    nn.linear_packed(x, w, "MXFP8_E4M3", residual=part[:, 3:67]).sum().backward()
    assert part.grad[:, 3:67].eq(1).all() and part.grad.count_nonzero() == 5 * 64
    far = torch.zeros(5, 64, dtype=torch.bfloat16, requires_grad=True)                      # a residual that lives on the CPU
    nn.linear_packed(x, w, "MXFP8_E4M3", residual=far).sum().backward()
    assert far.grad.device.type == "cpu" and far.grad.eq(1).all()


def test_no_gradient_is_lost():
    from mxq import nn
    x, w, bias, r = operands()
    plan = nn.dispatch(torch.tensor([[0], [1], [1], [0], [1]], dtype=torch.int32, device=DEV), 2)
    we, be = tuple(torch.stack((t, t)) for t in w), torch.stack((bias, bias))
    leaf = lambda t: t.clone().requires_grad_(True)  # noqa: E731
    calls = [
        ("for x", lambda: nn.linear_packed(leaf(x), w, "MXFP8_E4M3")),
        ("for x", lambda: nn.linear_packed(leaf(x) * 2, w, "MXFP8_E4M3", residual=leaf(r))),
        ("for bias", lambda: nn.linear_packed(x, w, "MXFP8_E4M3", bias=leaf(bias), out=torch.float32)),
        ("for x", lambda: nn.experts_packed(leaf(x), we, "MXFP8_E4M3", plan)),
        ("for bias", lambda: nn.experts_packed(x, we, "MXFP8_E4M3", plan, bias=leaf(be), out=torch.float16)),
    ]
    for text, call in calls:
        y = call()                                        # the values are there
        assert y.requires_grad
        with pytest.raises(RuntimeError, match=f"inference only.*{text}"):
            y.float().sum().backward()
        with torch.no_grad():
            z = call()
        assert not z.requires_grad and torch.equal(y.detach(), z)
        with torch.inference_mode():
            assert torch.equal(call(), z)


def raises_forward(calls):
    for call in calls:
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises((RuntimeError, NotImplementedError), match="(?i)forward"):
                call()


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


def test_forward_mode_raises():
    from mxq import nn
    x, w, bias, r = operands()
    want = nn.linear_packed(x, w, "MXFP8_E4M3")
    with forward_ad.dual_level():
        raises_forward((lambda: nn.linear_packed(dual(x), w, "MXFP8_E4M3"), lambda: nn.linear_packed(x, w, "MXFP8_E4M3", bias=dual(bias)),
                        lambda: nn.linear_packed(x, w, "MXFP8_E4M3", residual=dual(r))))
        assert torch.equal(nn.linear_packed(x, w, "MXFP8_E4M3"), want)                      # no tangent: as ever


def test_forward_mode_raises_in_routing():
    from mxq import nn
    logits = torch.randn(4, 8, device=DEV)
    weights, experts = nn.route(logits, 2)
    plan, z = nn.dispatch(experts, 8), torch.randn(8, 16, device=DEV)
    with forward_ad.dual_level():
        raises_forward((lambda: nn.route(dual(logits), 2), lambda: nn.combine(dual(z), weights, plan),
                        lambda: nn.combine(z, dual(weights), plan), lambda: nn.combine(z, weights, plan, residual=dual(z[:4]))))
        assert torch.equal(nn.route(logits, 2)[0], weights)
