"""nn.route's groups from their definition, row by row in float64: a group's value is its largest choice value, or the sum of its two
largest scores + bias, in which a masked expert has the score 0; the best groups with an expert to choose are kept."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPES = [(8, 4, 2), (64, 8, 3), (256, 8, 4), (96, 4, 1), (40, 5, 2), (60, 3, 3), (128, 32, 7), (1024, 16, 4), (12, 12, 5), (6, 3, 1)]


def route64(logits, k, score, groups, keep, by, bias=None):
    """(experts, the smallest distance between two values of groups or chosen experts that differ)"""
    T, E = logits.shape
    l, run = logits.double(), E // groups
    s = torch.where(l == -math.inf, torch.zeros_like(l), torch.sigmoid(l) if score == "sigmoid" else torch.softmax(l, -1))
    v = s + (bias.double() if bias is not None else 0)
    order = l if bias is None else v
    out, margin = torch.full((T, k), -1, dtype=torch.int32), math.inf
    for t in range(T):
        live = [e for e in range(E) if l[t, e] > -math.inf]
        value = {}
        for g in {e // run for e in live}:
            if by == "top2":
                value[g] = sum(sorted(v[t, g * run:(g + 1) * run].tolist())[-2:])
            else:
                value[g] = max(float(order[t, e]) for e in live if e // run == g)
        kept = sorted(value, key=lambda g: (-value[g], g))[:keep]
        chosen = sorted((e for e in live if e // run in kept), key=lambda e: (-float(order[t, e]), e))[:k]
        out[t, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
        for vs in (sorted(value.values()), sorted(float(order[t, e]) for e in live)):
            margin = min([margin] + [b - a for a, b in zip(vs, vs[1:]) if b > a])
    return out, margin


def spread(T, E, score, g):
    """Logits whose scores, and the sums of two of them, are apart by more than float32's rounding: distinct multiples of a
    fine step."""
    if score == "sigmoid":
        s = (torch.stack([torch.randperm(8 * E, generator=g)[:E] for _ in range(T)]).double() + 0.5) / (8 * E)
        return torch.log(s / (1 - s)).float()
    return 0.6 * torch.randn(T, E, generator=g)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,keep", SHAPES)
def test_groups_by_scores(score, E, groups, keep):
    from mxq import nn
    g = torch.Generator().manual_seed(E * 7 + groups)
    logits = spread(40, E, score, g)
    logits[20:] = torch.where(torch.rand(20, E, generator=g) < 0.4, torch.tensor(-math.inf), logits[20:])
    k = min(4, keep * (E // groups))
    for by in ("max", "top2"):
        for bias in (None, 0.3 * torch.randn(E, generator=g)):
            compared = 0
            got = nn.route(logits.to(DEV), k, score=score, groups=groups, keep=keep, group_score=by,
                           bias=None if bias is None else bias.to(DEV))[1].cpu()
            for t in range(40):                          # rows whose values are not nearer than float32 tells apart
                want, margin = route64(logits[t:t + 1], k, score, groups, keep, by, bias)
                if margin > 1e-6:
                    compared += 1
                    assert torch.equal(got[t:t + 1], want), (by, t, margin)
            assert compared >= 20, compared


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,keep", SHAPES)
def test_a_bias_of_zeros_changes_no_group(score, E, groups, keep):
    """Bit for bit, ties and all (logits of few values, and wide ones whose scores underflow): the same groups are kept."""
    from mxq import nn
    g = torch.Generator().manual_seed(E + 1)
    for logits in (2 * torch.randn(50, E, generator=g), torch.randint(-2, 3, (50, E), generator=g).float(),
                   60 * torch.randn(50, E, generator=g)):
        every = min(32, keep * (E // groups))
        kw = dict(score=score, groups=groups, keep=keep, group_score="top2")
        a = nn.route(logits.to(DEV), every, **kw)[1]
        b = nn.route(logits.to(DEV), every, bias=torch.zeros(E, device=DEV), **kw)[1]
        run = E // groups
        for x, y in zip((a // run).tolist(), (b // run).tolist()):
            if every == keep * run:                      # all experts of the kept groups
                assert sorted(x) == sorted(y)
            else:                                        # the best ones, which saturated scores may order otherwise
                assert set(x) == set(y) or logits.abs().max() > 20


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masking_does_not_raise_a_group(score):
    from mxq import nn
    inf = math.inf
    kw = dict(score=score, groups=2, keep=1, group_score="top2")
    rows = torch.tensor([[6, -9, -1.2, -1.2], [10, -5, 2, 2], [-1, -1, -0.8, -0.8], [-1, -inf, -0.8, -0.8],
                         [-inf, -inf, -50, -inf], [-inf, -3, -inf, -inf]]).to(DEV)
    for bias in (None, torch.zeros(4, device=DEV)):
        experts = nn.route(rows, 2, bias=bias, **kw)[1].tolist()
        if score == "sigmoid":                            # 0.9976 against 0.463; 1.0066 against 1.762
            assert experts[:2] == [[0, 1], [2, 3]]
        else:                                             # softmax: 6 and 10 outweigh the rest
            assert experts[:2] == [[0, 1], [0, 1]]
        assert experts[2:] == [[2, 3], [2, 3], [2, -1], [1, -1]]
    # negative choice values: -0.3 and -0.1 against two of -0.25, one of which is then masked and counts as its bias alone
    bias = torch.tensor([-0.8, -0.6, -0.75, -0.75], device=DEV)
    same = torch.zeros(1, 4, device=DEV)
    masked = torch.tensor([[0, 0, 0, -inf]], device=DEV)
    if score == "sigmoid":
        assert nn.route(same, 2, bias=bias, **kw)[1].tolist() == [[1, 0]]
        assert nn.route(masked, 2, bias=bias, **kw)[1].tolist() == [[1, 0]]
        low = torch.tensor([-0.8, -0.6, -0.75, -inf], device=DEV)                    # a bias that takes an expert out
        assert nn.route(same, 2, bias=low, **kw)[1].tolist() == [[1, 0]]
