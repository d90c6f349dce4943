"""Rows of logits that have no scores: nn.route's weights and their gradient are NaN there, whatever chooses the experts, and the
token's result shows it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("E", [4, 33, 256])
@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("how", [{}, {"renormalize": True}, {"groups": 1, "bias": True}, {"groups": 1, "bias": True, "renormalize": True}])
def test_softmax_without_scores(dtype, E, value, how):
    from mxq import nn
    g = torch.Generator().manual_seed(E)
    logits = torch.randn(6, E, generator=g).to(DEV, dtype)
    logits[2, E // 2] = value
    logits[4] = value
    how = dict(how, bias=torch.randn(E, generator=g).to(DEV) if how.get("bias") else None)
    clean = logits.clone()
    clean[2], clean[4] = 0, 0
    a = logits.clone().requires_grad_(True)
    w, x = nn.route(a, 3, score="softmax", **how)
    w0, x0 = nn.route(clean, 3, score="softmax", **how)
    rows = torch.tensor([0, 1, 3, 5], device=DEV)
    assert w[[2, 4]].isnan().all()
    assert torch.equal(w[rows], w0[rows]) and torch.equal(x[rows], x0[rows])
    grad, = torch.autograd.grad(w, a, torch.ones_like(w))
    assert grad[[2, 4]].isnan().all() and torch.isfinite(grad[rows]).all()

    plan = nn.dispatch(x, E)
    z = torch.randn(18, 8, generator=g).to(DEV)
    y = nn.combine(z, w.detach(), plan)
    assert y[[2, 4]].isnan().all() and torch.isfinite(y[rows]).all()


def test_sigmoid_of_inf_is_one():
    """+Inf is a score of 1 under sigmoid, with and without a bias."""
    from mxq import nn
    logits = torch.zeros(2, 8, device=DEV)
    logits[1, 5] = math.inf
    for bias in (None, torch.zeros(8, device=DEV)):
        w, x = nn.route(logits, 2, score="sigmoid", bias=bias)
        assert x.tolist() == [[0, 1], [5, 0]] and w.tolist() == [[0.5, 0.5], [1.0, 0.5]]
