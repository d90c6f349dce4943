"""nn.route, nn.dispatch, nn.combine and their gradients against float64 row by row: ties, masked experts, rows without any,
NaN, groups of every shape, strided rows, one token to many, one expert to 1024; gradients against the formula and against
differences; and MXExperts, which runs them together."""
import math

import pytest
import torch

from _feedforward import assert_close, decode, dispatch64, product64, random_pair, route64, route_backward64

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def check_route(logits, k, what="", **kw):
    """Whole choices equal, weights within 2^-18 of their size (exp, the sum of up to 1024 and two divisions in
    float32) plus what an exp that underflows loses."""
    from mxq import nn
    ref = {"score": "softmax", **{n: v for n, v in kw.items() if n != "group_score"}}
    W, X, margin = route64(logits, k, top2=kw.get("group_score") == "top2", **ref)
    if kw.get("bias") is not None:
        assert margin > 1e-5, f"{what}: the inputs come too near a tie ({margin:.2g}) for float32"
    dev = {n: v.to(DEV) if isinstance(v, torch.Tensor) else v for n, v in kw.items()}
    w, x = nn.route(logits.to(DEV), k, **dev)
    assert w.dtype == torch.float32 and x.dtype == torch.int32
    assert torch.equal(x.cpu(), X), what
    w = w.cpu().double()
    assert torch.equal(w.isnan(), W.isnan()), what
    off = (w - W).abs()[~W.isnan()]
    assert (off <= 2.0 ** -18 * W[~W.isnan()] + 1e-30).all(), f"{what}: {float(off.max())}"


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E", [1, 5, 32, 33, 64, 100, 128, 256, 384, 1024])
def test_route(score, dtype, E):
    g = gen(E)
    for T in (1, 6):
        logits = (2 * torch.randn(T, E, generator=g)).to(dtype)
        for k in sorted({1, min(3, E), min(8, E), min(32, E)}):
            check_route(logits, k, f"{E} {k}", score=score, renormalize=k % 2 == 1, scale=1.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,keep", [(8, 4, 2), (64, 8, 3), (256, 8, 4), (96, 4, 1), (40, 5, 2), (60, 3, 3), (128, 32, 7),
                                           (1024, 16, 4), (12, 12, 5)])
def test_groups(score, E, groups, keep):
    g = gen(E + groups)
    logits = 2 * torch.randn(5, E, generator=g)
    k = min(4, keep * (E // groups))
    for by in ("max", "top2"):
        check_route(logits, k, f"{E} {groups} {by}", score=score, groups=groups, keep=keep, group_score=by)
        # choice values 0.37 apart and more: no two sums of them meet in float32
        bias = 0.37 * torch.randperm(E, generator=g).float() + 0.01 * torch.rand(E, generator=g)
        check_route(logits, k, f"{E} {groups} {by} bias", score=score, groups=groups, keep=keep, group_score=by, bias=bias,
                    renormalize=True)


def test_ties_and_masks():
    """Equal logits go to the lowest index, -0 and 0 are equal, -Inf is never chosen, an empty row has no expert."""
    g = gen(3)
    logits = torch.randint(-1, 2, (40, 48), generator=g).float()
    logits[3] = 0.0
    logits[4] = torch.where(torch.arange(48) % 2 == 0, torch.tensor(-0.0), torch.tensor(0.0))
    logits[5, 3:] = -math.inf
    logits[6] = -math.inf
    logits[7, 10] = math.nan
    logits[8] = math.nan
    logits[9] = torch.finfo(torch.float32).min
    for score in ("softmax", "sigmoid"):
        for groups, keep in ((1, 1), (4, 2), (6, 5)):
            check_route(logits, 5, f"{score} {groups}", score=score, groups=groups, keep=keep, renormalize=True)
            check_route(logits, 5, f"{score} {groups} top2", score=score, groups=groups, keep=keep, group_score="top2")
    big = torch.tensor([[1e4, -1e4, 80.0, -80.0, 0.0, 1e4]])
    for score in ("softmax", "sigmoid"):
        check_route(big.clamp(-700, 700), 6, score=score)


def test_route_layouts():
    from mxq import nn
    g = gen(5)
    wide = torch.randn(30, 300, generator=g).to(DEV)
    for part in (wide[:, :128], wide[:, 3:131], wide[::2, 4:132], wide.T[:128].T[:5]):
        for a, b in zip(nn.route(part, 4), nn.route(part.contiguous(), 4)):
            assert torch.equal(a, b)
    cols = torch.randn(128, 30, generator=g).to(DEV).T                  # not contiguous along the experts
    for a, b in zip(nn.route(cols, 4), nn.route(cols.contiguous(), 4)):
        assert torch.equal(a, b)
    w, x = nn.route(torch.empty(0, 16, device=DEV), 2)
    assert w.shape == x.shape == (0, 2)
    cpu = nn.route(wide.cpu(), 3)
    assert cpu[0].device.type == "cpu" and torch.equal(cpu[1], nn.route(wide, 3)[1].cpu())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("E,k", [(1, 1), (8, 2), (64, 6), (100, 32), (1024, 8)])
def test_route_backward(dtype, score, renormalize, E, k):
    """Against the formula: terms of at most |g| / S and |g| s, each with a few roundings of float32 (2^-18 of the
    largest), then the logits' own type."""
    from mxq import nn
    g = gen(E + k)
    logits = torch.randn(9, E, generator=g).to(dtype)
    if E > 2 * k:
        logits[2, 1::2] = -math.inf
    grad = torch.randn(9, k, generator=g)
    _, x = nn.route(logits.to(DEV), k, score=score)
    got = nn.route_backward(grad.to(DEV), logits.to(DEV), x, score=score, renormalize=renormalize, scale=1.5)
    assert got.dtype == dtype and got.shape == logits.shape
    want = route_backward64(grad.to(DEV), logits.to(DEV), x, score, renormalize, 1.5)
    s = torch.softmax(logits.to(DEV).double(), -1) if score == "softmax" else torch.sigmoid(logits.to(DEV).double())
    total = s.gather(1, x.long()).sum(1, keepdim=True) if renormalize else torch.ones(9, 1, device=DEV)
    size = 1.5 * grad.abs().amax(1, keepdim=True).to(DEV).double() * k / total
    assert_close(got, want, 2.0 ** -18 * size * s.clamp_max(1) + 1e-30, dtype, f"{score} {E}")


def test_route_backward_holes():
    """Places without an expert take no part; a NaN in a row reaches that row's gradient only."""
    from mxq import nn
    logits = torch.randn(4, 16, generator=gen(7)).to(DEV)
    logits[1] = -math.inf
    logits[2, 2:] = -math.inf
    w, x = nn.route(logits, 4, renormalize=True)
    assert (x[1] == -1).all() and (x[2, 2:] == -1).all()
    grad = torch.randn(4, 4, generator=gen(8)).to(DEV)
    got = nn.route_backward(grad, logits, x, renormalize=True)
    want = route_backward64(grad[[0, 2, 3]], logits[[0, 2, 3]], x[[0, 2, 3]], "softmax", True, 1.0)
    assert (got[1] == 0).all() and (got[[0, 2, 3]] - want).abs().max() < 1e-5
    logits[3, 5] = math.nan
    bad = nn.route_backward(grad, logits, x, renormalize=True)
    assert bad[3].isnan().all() and torch.equal(bad[:3], got[:3])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_route_differences(score, renormalize):
    """autograd through route against central differences of its own weights: step h = 2^-5 costs h^2 / 6 of the third
    derivative (below 1 for weights up to 2: 1.7e-4 a weight) and the float32 weights 2^-23 / h; 4 weights a row."""
    from mxq import nn
    g = gen(9)
    logits = (torch.randn(3, 8, generator=g) * 0.5 + torch.arange(8) * 0.7).to(DEV)   # the choice does not change within h
    coef = torch.randn(3, 4, generator=g).to(DEV)
    kw = dict(score=score, renormalize=renormalize, scale=1.0)
    a = logits.clone().requires_grad_(True)
    w, x = nn.route(a, 4, **kw)
    (w * coef).sum().backward()
    h = 2.0 ** -5
    for t in range(3):
        for e in range(8):
            up, down = logits.clone(), logits.clone()
            up[t, e] += h
            down[t, e] -= h
            sides = []
            for moved in (up, down):                                  # the same experts, maybe in another order
                wm, xm = nn.route(moved, 4, **kw)
                assert torch.equal(xm.sort(1).values, x.sort(1).values)
                every = torch.zeros(3, 8, device=DEV).scatter_(1, xm.long(), wm)
                sides.append(every.gather(1, x.long()).double())
            diff = float(((sides[0] - sides[1]) * coef).sum()) / (2 * h)
            assert abs(diff - float(a.grad[t, e])) < 4 * 4 * (1.7e-4 + 2.0 ** -23 / h)


# ----------------------------------------------------------------------------------------------- dispatch
@pytest.mark.parametrize("T,k,E", [(0, 2, 4), (1, 1, 1), (3, 2, 7), (31, 3, 64), (100, 8, 256), (513, 1, 1024), (3000, 8, 33),
                                   (9000, 8, 128), (70001, 4, 17)])
def test_dispatch(T, k, E):
    from mxq import nn
    g = gen(T + E)
    for low, high in ((0, E), (-2, E + 3), (E - 1, E), (-1, 0)):
        experts = torch.randint(low, high, (T, k), generator=g).int()
        want = dispatch64(experts, E)
        got = nn.dispatch(experts.to(DEV), E)
        for name, a, b in zip(got._fields, got, want):
            assert torch.equal(a.cpu(), b), (name, T, k, E, low)


# ------------------------------------------------------------------------------------------------ combine
def plan_with_holes(T, k, E, g):
    from mxq import nn
    return nn.dispatch(torch.randint(-1, E, (T, k), generator=g).int().to(DEV), E)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,N", [(1, 1, 1), (5, 2, 33), (64, 6, 256), (17, 9, 1000), (3, 8, 4100), (700, 4, 72), (2, 33, 24)])
def test_combine(dtype, T, k, N):
    """k products and sums in float32: (k + 1) 2^-23 of the absolute sum; the residual one rounding more."""
    from mxq import nn
    g = gen(T + k + N)
    plan = plan_with_holes(T, k, 6, g)
    z = torch.randn(T * k, N, generator=g).to(DEV, dtype)
    z[int(plan.offsets[-1]):] = math.nan                                 # rows that no slot has are not read
    weights = torch.randn(T, k, generator=g).to(DEV)
    at = plan.where.long()
    rows = torch.where(at[..., None] >= 0, z[at.clamp_min(0)].double(), torch.zeros((), dtype=torch.float64, device=DEV))
    want = (weights.double()[..., None] * rows).sum(1)
    size = (weights.double()[..., None] * rows).abs().sum(1)
    y = nn.combine(z, weights, plan)
    assert y.dtype == dtype
    assert_close(y, want, (k + 1) * 2.0 ** -23 * size, dtype)
    wide = torch.randn(T, N + 9, generator=g).to(DEV, dtype)
    for r in (wide[:, :N].contiguous(), wide[:, 5:5 + N]):
        assert_close(nn.combine(z, weights, plan, residual=r), want + r.double(),
                     (k + 2) * 2.0 ** -23 * (size + r.double().abs()), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,N", [(1, 1, 1), (5, 2, 33), (64, 6, 256), (17, 9, 1000), (3, 8, 4100), (700, 4, 72), (2, 33, 24),
                                   (6, 3, 2048), (4, 5, 512)])
def test_combine_backward(dtype, T, k, N):
    from mxq import nn
    g = gen(T + k + N + 1)
    plan = plan_with_holes(T, k, 6, g)
    z, dy = torch.randn(T * k, N, generator=g).to(DEV, dtype), torch.randn(T, N, generator=g).to(DEV, dtype)
    weights = torch.randn(T, k, generator=g).to(DEV)
    dz, dw = nn.combine_backward(dy, z, weights, plan)
    order, at = plan.order.long(), plan.where.long()
    live = order >= 0
    want = torch.zeros(T * k, N, dtype=torch.float64, device=DEV)
    want[live] = weights.double().flatten()[order[live], None] * dy.double()[order[live] // k]
    assert_close(dz, want, torch.zeros_like(want), dtype, "dz")
    rows = torch.where(at[..., None] >= 0, z[at.clamp_min(0)].double(), torch.zeros((), dtype=torch.float64, device=DEV))
    prod = dy.double()[:, None] * rows
    assert_close(dw, prod.sum(-1), (N + 1) * 2.0 ** -23 * prod.abs().sum(-1), torch.float32, "dw")
    wide = torch.randn(T, N + 3, generator=g).to(DEV, dtype)[:, 1:1 + N]
    for a, b in zip(nn.combine_backward(wide, z, weights, plan), nn.combine_backward(wide.contiguous(), z, weights, plan)):
        assert torch.equal(a, b)


def test_combine_differences():
    """combine is linear in each argument: differences with step 1 are exact up to float32's rounding of y (|y| < 16)."""
    from mxq import nn
    g = gen(11)
    plan = plan_with_holes(4, 3, 5, g)
    z, weights = torch.randn(12, 10, generator=g).to(DEV), torch.randn(4, 3, generator=g).to(DEV)
    r, coef = torch.randn(4, 10, generator=g).to(DEV), torch.randn(4, 10, generator=g).to(DEV)
    leaves = [t.clone().requires_grad_(True) for t in (z, weights, r)]
    (nn.combine(leaves[0], leaves[1], plan, residual=leaves[2]) * coef).sum().backward()
    base = [z, weights, r]
    for which, leaf in enumerate(leaves):
        for i in range(leaf.numel()):
            up = [t.clone() for t in base]
            up[which].view(-1)[i] += 1
            diff = ((nn.combine(up[0], up[1], plan, residual=up[2]) - nn.combine(*base[:2], plan, residual=base[2])).double()
                    * coef.double()).sum()
            assert abs(float(diff) - float(leaf.grad.view(-1)[i])) < 10 * 16 * 2.0 ** -22


# ------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("fmt", ["MXFP8_E4M3", "MXFP6_E2M3", "MXFP4"])
@pytest.mark.parametrize("T", [1, 30, 500])
def test_experts_layer(fmt, T):
    """MXExperts is its operators one after the other, bit for bit, and from the packed hidden rows on within their bounds of
    float64 on its packed weights (the down products' in bfloat16, then the weighted sum's)."""
    from mxq import nn
    g = gen(13)
    E, k, H, F = 8, 3, 96, 160
    up, down = torch.randn(E, 2 * F, H, generator=g) / H ** 0.5, torch.randn(E, H, F, generator=g) / F ** 0.5
    layer = nn.MXExperts(up.to(DEV), down.to(DEV), fmt)
    x = torch.randn(T, H, generator=g).to(DEV, torch.bfloat16)
    logits = torch.randn(T, E, generator=g).to(DEV)
    if T > 1:
        logits[1] = -math.inf                                           # a padded token
    weights, experts = nn.route(logits, k, renormalize=True)
    y = layer(x, weights, experts, residual=x)
    assert y.shape == x.shape and y.dtype == x.dtype

    plan = nn.dispatch(experts, E)
    wu, wd = (layer.up_codes, layer.up_scales), (layer.down_codes, layer.down_scales)
    h = nn.experts_packed(x, wu, layer.up_fmt, plan, activation="swiglu", out="MXFP8_E4M3")
    z = nn.experts_packed(h, wd, layer.down_fmt, plan, gather=False, out=torch.bfloat16)
    assert torch.equal(y, nn.combine(z, weights, plan, residual=x))

    rows, at = decode(h, "MXFP8_E4M3"), plan.where.long()
    down64 = decode(wd, layer.down_fmt)
    zs, room = torch.zeros(T, k, H, dtype=torch.float64, device=DEV), torch.zeros(T, k, H, dtype=torch.float64, device=DEV)
    for t in range(T):
        for j in range(k):
            if at[t, j] >= 0:
                v, b = product64(rows[at[t, j]][None], down64[int(experts[t, j])])
                zs[t, j], room[t, j] = v[0], b[0] + 2.0 ** -8 * (v[0].abs() + b[0])
    w64 = weights.double()[..., None]
    want, bound = (w64 * zs).sum(1) + x.double(), (w64.abs() * room).sum(1)
    assert_close(y, want, bound + (k + 2) * 2.0 ** -23 * ((w64 * zs).abs().sum(1) + x.double().abs()), torch.bfloat16, fmt)
    if T > 1:
        assert torch.equal(y[1], x[1])


def test_experts_layer_gradient():
    """The router's gradient through the packed experts is combine's and route's."""
    from mxq import nn
    g = gen(17)
    E, k, H, F, T = 6, 2, 64, 64, 20
    layer = nn.MXExperts(torch.randn(E, 2 * F, H, generator=g).to(DEV) / 8, torch.randn(E, H, F, generator=g).to(DEV) / 8)
    x, router = torch.randn(T, H, generator=g).to(DEV), torch.randn(E, H, generator=g).to(DEV).requires_grad_(True)
    logits = x @ router.T
    weights, experts = nn.route(logits, k, renormalize=True)
    y = layer(x, weights, experts)
    dy = torch.randn(T, H, generator=g).to(DEV)
    y.backward(dy)
    plan = nn.dispatch(experts, E)
    pair = lambda n: (getattr(layer, n + "_codes"), getattr(layer, n + "_scales"))  # noqa: E731
    h = nn.experts_packed(x, pair("up"), layer.up_fmt, plan, activation="swiglu", out="MXFP8_E4M3")
    z = nn.experts_packed(h, pair("down"), layer.down_fmt, plan, gather=False, out=torch.float32)
    _, dw = nn.combine_backward(dy, z, weights.detach(), plan)
    dl = nn.route_backward(dw, logits.detach(), experts, renormalize=True)
    assert torch.allclose(router.grad, dl.T @ x, rtol=0, atol=1e-4 * float(router.grad.abs().max()))


def test_refusals():
    from mxq import nn
    l = torch.randn(4, 12, device=DEV)
    w, x = nn.route(l, 2)
    plan = nn.dispatch(x, 12)
    z = torch.randn(8, 16, device=DEV)
    cases = [
        ("2-D float32", lambda: nn.route(l.double(), 2)), ("2-D float32", lambda: nn.route(l[0], 2)),
        ("k must be", lambda: nn.route(l, 0)), ("k must be", lambda: nn.route(l, 13)), ("k must be", lambda: nn.route(l, 2.0)),
        ("score must be", lambda: nn.route(l, 2, score="relu")), ("score must be", lambda: nn.route(l, 2, group_score="mean")),
        ("cannot keep", lambda: nn.route(l, 2, groups=5)), ("cannot keep", lambda: nn.route(l, 2, groups=4, keep=5)),
        ("bias", lambda: nn.route(l, 2, bias=torch.zeros(11, device=DEV))),
        ("1024 experts", lambda: nn.route(torch.zeros(1, 1025, device=DEV), 2)),
        ("must be 4 x k", lambda: nn.route_backward(w[:3], l, x)), ("int32", lambda: nn.route_backward(w, l, x.long())),
        ("n_experts", lambda: nn.dispatch(x, 0)), ("n_experts", lambda: nn.dispatch(x, 1025)),
        ("int32", lambda: nn.dispatch(x.long(), 12)),
        ("do not match", lambda: nn.combine(z, w[:, :1], plan)), ("z has", lambda: nn.combine(z[:7], w, plan)),
        ("z must be", lambda: nn.combine(z.double(), w, plan)),
        ("residual", lambda: nn.combine(z, w, plan, residual=torch.zeros(4, 15, device=DEV))),
        ("dy must be", lambda: nn.combine_backward(z[:3], z, w, plan)),
        ("gate_up", lambda: nn.MXExperts(torch.zeros(2, 10, 8), torch.zeros(2, 8, 4))),
        ("activation", lambda: nn.MXExperts(torch.zeros(2, 8, 8), torch.zeros(2, 8, 4), activation="silu")),
    ]
    for text, call in cases:
        with pytest.raises(ValueError, match=text):
            call()
    layer = nn.MXExperts(torch.randn(2, 64, 32, device=DEV), torch.randn(2, 32, 32, device=DEV))
    with pytest.raises(ValueError, match="must be"):
        layer(torch.zeros(3, 32, device=DEV), torch.zeros(2, 1, device=DEV), torch.zeros(2, 1, device=DEV, dtype=torch.int32))
