"""The feed-forward's calls as a serving program makes them: captured in a CUDA graph and replayed on other inputs, and from two
streams at the same time. The same bits as eager calls, one after the other. And the sums' exactness as a whole."""
import pytest
import torch

from _feedforward import decode, random_pair

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8 = "MXFP8_E4M3"


def gen(seed):
    return torch.Generator().manual_seed(seed)


def captured(call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


@pytest.mark.parametrize("M", [1, 24, 200, 900])
@pytest.mark.parametrize("fmt", [F8, "MXFP4", "MXFP6_E3M2"])
def test_a_captured_chain(M, fmt):
    """Floats packed in the call, a packed product behind it, a residual: launches that start before the one ahead has ended."""
    from mxq import nn
    g = gen(M)
    x = torch.randn(M, 1000, generator=g).to(DEV, torch.bfloat16)
    up, down = random_pair((2 * 384, 1000), fmt, g, DEV), random_pair((1000, 384), F8, g, DEV)
    up, down = (up[0], up[1] - 6), (down[0], down[1] - 6)

    def call():
        h = nn.linear_packed(x, up, fmt, activation="swiglu", out=F8)
        return nn.linear_packed(h, down, F8, residual=x)
    graph, out = captured(call)
    for i in range(4):
        x.copy_(torch.randn(M, 1000, generator=g))
        graph.replay()
        if i == 2:
            graph.replay()                                # twice without a wait
        got = out.clone()
        assert torch.equal(got, call())


@pytest.mark.parametrize("T", [1, 16, 700])
def test_a_captured_layer(T):
    """Router, dispatch, both products by expert and the weighted sum; the choice changes from replay to replay."""
    from mxq import nn
    g = gen(T + 1)
    E, k, H, F = 8, 2, 128, 192
    layer = nn.MXExperts(torch.randn(E, 2 * F, H, generator=g).to(DEV) / 8, torch.randn(E, H, F, generator=g).to(DEV) / 8)
    router = torch.randn(H, E, generator=g).to(DEV)
    x = torch.randn(T, H, generator=g).to(DEV)

    def call():
        weights, experts = nn.route(x @ router, k, score="sigmoid", groups=4, keep=2, group_score="top2", renormalize=True)
        return layer(x, weights, experts, residual=x), experts
    graph, (y, experts) = captured(call)
    seen = []
    for _ in range(4):
        x.copy_(torch.randn(T, H, generator=g))
        graph.replay()
        got, chosen = y.clone(), experts.clone()
        want, again = call()
        assert torch.equal(got, want) and torch.equal(chosen, again)
        seen.append(chosen)
    assert any(not torch.equal(seen[0], s) for s in seen[1:])


def test_a_captured_dispatch_of_many_slots():
    from mxq import nn
    g = gen(3)
    e = torch.zeros(30000, 4, dtype=torch.int32, device=DEV)                                # two launches
    graph, plan = captured(lambda: nn.dispatch(e, 64))
    for _ in range(3):
        e.copy_(torch.randint(-1, 64, (30000, 4), generator=g))
        graph.replay()
        for a, b in zip([t.clone() for t in plan], nn.dispatch(e, 64)):
            assert torch.equal(a, b)


def test_two_streams():
    """Few rows over clusters beside pairs of CTAs with all of an SM's tensor memory, on operands that both streams read."""
    from mxq import nn
    g = gen(5)
    w = random_pair((1536, 2048), F8, g, DEV)
    xs = [random_pair((M, 2048), F8, g, DEV) for M in (1, 700, 33, 300, 16, 2000)]
    want = [nn.linear_packed(x, w, F8, out=torch.float32) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                for x in (xs if i == 0 else xs[::-1]):
                    got[i].append(nn.linear_packed(x, w, F8, out=torch.float32))
    torch.cuda.synchronize()
    for i, order in enumerate((want, want[::-1])):
        for j, y in enumerate(got[i]):
            assert torch.equal(y, order[j % len(want)]), (i, j)


@pytest.mark.parametrize("M", [16, 300])
@pytest.mark.parametrize("K", [2048, 8192])
def test_the_sums_are_float32(M, K):
    """The norm of the error of float32 sums of K / 32 additions, each of which may lose 2^-23 of the running sum: with random
    signs that grows as the square root of its length, so the losses sum to 2/3 K/32 2^-23 of the result. (An accumulator of 16 bits
    is beyond that by two orders.)"""
    from mxq import nn
    g = gen(K + M)
    x, w = random_pair((M, K), F8, g, DEV), random_pair((512, K), F8, g, DEV)
    y = nn.linear_packed(x, w, F8, out=torch.float32).double()
    exact = decode(x, F8) @ decode(w, F8).T
    assert (y - exact).norm() <= 2 / 3 * (K / 32) * 2.0 ** -23 * exact.norm()
