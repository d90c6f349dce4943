"""nn.linear_packed and nn.experts_packed against float64: sizes on both sides of every tile and block edge, every pair of
formats, activations, output types, residuals, masked and special values, plans with empty experts and left-out slots.
Bounds are those of _feedforward.product64 (float32 sums) plus the output's own rounding."""
import math

import pytest
import torch

from _feedforward import FORMATS, assert_close, assert_packed, decode, product64, random_pair

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator().manual_seed(seed)


def check(x, xf, w, wf, bias=None, activation=None, residual=None, out=torch.float32, what=""):
    from mxq import nn
    y = nn.linear_packed(x, w, wf, x_fmt=xf, bias=bias, activation=activation, residual=residual, out=out)
    want, bound = product64(decode(x, xf), decode(w, wf), bias, activation)
    if isinstance(out, str):
        return assert_packed(y, want, bound, out, what)
    assert y.dtype == out and y.shape == want.shape
    if residual is not None:
        want = want + residual.double()
        bound = bound + 2.0 ** -23 * want.abs()
    assert_close(y, want, bound, out, what)


ROWS = [1, 2, 15, 16, 17, 32, 33, 64, 65, 129, 255, 257, 600]


@pytest.mark.parametrize("M", ROWS)
def test_rows(M):
    """Every row count at which the tiles change, columns and K no multiple of a tile."""
    g = gen(M)
    for N, K in ((1, 32), (130, 96), (257, 640), (514, 160)):
        x, w = random_pair((M, K), "MXFP8_E4M3", g, DEV), random_pair((N, K), "MXFP8_E4M3", g, DEV)
        check(x, "MXFP8_E4M3", w, "MXFP8_E4M3", what=f"{M} x {N} x {K}")


@pytest.mark.parametrize("K", [1, 2, 16, 31, 33, 48, 100, 127, 128, 129, 160, 528, 1000, 2049, 4224])
def test_depths(K):
    """K that ends inside a block, a step of the products, a word of scales, a group of four steps."""
    g = gen(1000 + K)
    for M, N in ((3, 200), (300, 700)):
        for wf in ("MXFP8_E4M3", "MXFP6_E2M3") + (("MXFP4",) if K % 2 == 0 else ()):
            x, w = random_pair((M, K), "MXFP8_E5M2", g, DEV), random_pair((N, K), wf, g, DEV)
            check(x, "MXFP8_E5M2", w, wf, what=f"{M} x {N} x {K} {wf}")


@pytest.mark.parametrize("M", [5, 700])
@pytest.mark.parametrize("xf", sorted(FORMATS))
@pytest.mark.parametrize("wf", sorted(FORMATS))
def test_formats(M, xf, wf):
    g = gen(7)
    for K in (256, 288):
        x, w = random_pair((M, K), xf, g, DEV), random_pair((384, K), wf, g, DEV)
        check(x, xf, w, wf, what=f"{xf} {wf} {K}")


@pytest.mark.parametrize("M", [1, 40, 900])
@pytest.mark.parametrize("activation", [None, "relu", "gelu", "gelu_tanh", "silu", "swiglu", "geglu"])
def test_epilogue(M, activation):
    """Bias, activation, residual and every output type; widths that are and are not whole 16-byte rows and blocks."""
    g = gen(11)
    for N in (512, 356, 134):
        x, w = random_pair((M, 192), "MXFP8_E4M3", g, DEV, 1), random_pair((N, 192), "MXFP8_E4M3", g, DEV, 1)
        w = (w[0], w[1] - 4)                            # sums of a few units, where the activations bend
        F = N // 2 if activation in ("swiglu", "geglu") else N
        bias = torch.randn(N, generator=g).to(DEV)
        for out in (torch.float32, torch.bfloat16, torch.float16):
            r = torch.randn(M, F, generator=g).to(DEV, out)
            check(x, "MXFP8_E4M3", w, "MXFP8_E4M3", bias, activation, r, out, f"{N} {out}")
            wide = torch.randn(M, F + 7, generator=g).to(DEV, out)[:, 3:3 + F]      # rows apart, base unaligned
            check(x, "MXFP8_E4M3", w, "MXFP8_E4M3", None, activation, wide, out, f"{N} {out} strided residual")
        for out in sorted(FORMATS):
            if out == "MXFP4" and F % 2:
                continue
            check(x, "MXFP8_E4M3", w, "MXFP8_E4M3", bias, activation, None, out, f"{N} {out}")


@pytest.mark.parametrize("M", [3, 400])
def test_packed_floats(M):
    """A float x is packed by the rule of a packed output; strided rows, three dimensions, every type and format."""
    from mxq import nn
    g = gen(13)
    eye = torch.eye(96)
    one = (eye.to(torch.float8_e4m3fn).view(torch.uint8).to(DEV), torch.full((96, 3), 127, dtype=torch.uint8, device=DEV))
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        v = (torch.randn(M, 96, generator=g) * torch.exp2(torch.randint(-6, 6, (M, 1), generator=g))).to(DEV, dtype)
        v[0, :40] = 0
        for fmt in sorted(FORMATS):
            y = nn.linear_packed(v, one, "MXFP8_E4M3", x_fmt=fmt, out=torch.float32)     # the packed x's values
            e, m, emax, top = FORMATS[fmt]
            b = v.double().unflatten(-1, (3, 32))
            amax = b.abs().amax(-1, keepdim=True)
            X = torch.exp2((torch.frexp(amax)[1] - 1 - emax).clamp(-127, 127).double())
            z = (b / X).clamp(-top, top)
            step = torch.exp2(torch.floor(torch.log2(z.abs().clamp_min(2.0 ** (2 - 2 ** (e - 1))))) - m)
            want = (torch.round(z / step) * step * X).flatten(-2)                         # torch.round is to nearest even
            assert torch.equal(y.double(), want), (dtype, fmt)
        wide = torch.randn(M, 131, generator=g).to(DEV, dtype)
        assert torch.equal(nn.linear_packed(wide[:, 5:101], one, "MXFP8_E4M3"),
                           nn.linear_packed(wide[:, 5:101].contiguous(), one, "MXFP8_E4M3"))
        assert torch.equal(nn.linear_packed(wide.T[:96].T, one, "MXFP8_E4M3"),
                           nn.linear_packed(wide[:, :96].contiguous(), one, "MXFP8_E4M3"))
        three = v.view(1, M, 96)
        assert torch.equal(nn.linear_packed(three, one, "MXFP8_E4M3")[0], nn.linear_packed(v, one, "MXFP8_E4M3"))


def test_packed_floats_match_block_ocp():
    """The packing of floats is block.ocp's compact form."""
    from mxq import block, nn
    g = gen(14)
    v = torch.randn(70, 320, generator=g).to(DEV)
    w = random_pair((90, 320), "MXFP8_E4M3", g, DEV)
    for fmt in sorted(FORMATS):
        pair = block.ocp.quantize_packed(v, fmt, axis=-1)
        assert torch.equal(nn.linear_packed(v, w, "MXFP8_E4M3", x_fmt=fmt), nn.linear_packed(pair, w, "MXFP8_E4M3", x_fmt=fmt)), fmt


@pytest.mark.parametrize("M", [4, 300])
def test_special_values(M):
    """A NaN code, an Inf code, a NaN scale reach their row or column only; scales at both ends of E8M0 meet."""
    from mxq import nn
    g = gen(17)
    N, K = 320, 256
    x, w = random_pair((M, K), "MXFP8_E5M2", g, DEV), random_pair((N, K), "MXFP8_E4M3", g, DEV)
    clean = nn.linear_packed(x, w, "MXFP8_E4M3", x_fmt="MXFP8_E5M2", out=torch.float32)
    x[0][1, 7] = 0x7f                                   # NaN
    x[1][2, 3] = 255                                    # NaN scale
    w[0][9, 200] = 0x7f                                 # NaN
    w[1][10, 0] = 255
    y = nn.linear_packed(x, w, "MXFP8_E4M3", x_fmt="MXFP8_E5M2", out=torch.float32)
    nan = torch.zeros(M, N, dtype=torch.bool, device=DEV)
    nan[1], nan[2], nan[:, 9], nan[:, 10] = True, True, True, True
    assert torch.equal(y.isnan(), nan)
    assert torch.equal(y[~nan], clean[~nan])
    codes, scales = nn.linear_packed(x, w, "MXFP8_E4M3", x_fmt="MXFP8_E5M2", out="MXFP8_E4M3")
    bad = nan.unflatten(-1, (-1, 32)).any(-1)
    assert torch.equal(scales == 255, bad)
    assert (codes.unflatten(-1, (-1, 32))[bad] == 0).all()
    x[0][:] = 0x3c                                      # ones, one Inf
    x[0][0, 0] = 0x7c
    x[1][:] = 127
    w[0][:] = 0x38
    w[0][3, 0] = 0x80 | 0x38
    w[0][4, 0] = 0
    w[1][:] = 127
    y = nn.linear_packed(x, w, "MXFP8_E4M3", x_fmt="MXFP8_E5M2", out=torch.float32)
    assert y[0, 0] == math.inf and y[0, 3] == -math.inf and y[0, 4].isnan() and torch.isfinite(y[1:]).all()
    x[0][0, 0] = 0x3c
    x[1][:], w[1][:] = 254, 0                           # 2^127 and 2^-127
    w[0][3, 0] = 0x38
    w[0][4, 0] = 0x38
    assert (nn.linear_packed(x, w, "MXFP8_E4M3", x_fmt="MXFP8_E5M2", out=torch.float32) == K).all()


def test_empty_and_homes():
    """No rows; rows of zeros; CPU tensors come back to the CPU; another stream; misaligned codes."""
    from mxq import nn
    g = gen(19)
    w = random_pair((70, 64), "MXFP8_E4M3", g, DEV)
    none = (torch.empty(0, 64, dtype=torch.uint8, device=DEV), torch.empty(0, 2, dtype=torch.uint8, device=DEV))
    assert nn.linear_packed(none, w, "MXFP8_E4M3").shape == (0, 70)
    x = random_pair((9, 64), "MXFP8_E4M3", g, DEV)
    y = nn.linear_packed(x, w, "MXFP8_E4M3")
    home = nn.linear_packed(tuple(t.cpu() for t in x), tuple(t.cpu() for t in w), "MXFP8_E4M3")
    assert home.device.type == "cpu" and torch.equal(home, y.cpu())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = nn.linear_packed(x, w, "MXFP8_E4M3")
    side.synchronize()
    assert torch.equal(y, z)
    odd = torch.empty(9 * 64 + 5, dtype=torch.uint8, device=DEV)[5:].view(9, 64).copy_(x[0])
    scales = torch.empty(9 * 2 + 3, dtype=torch.uint8, device=DEV)[3:].view(9, 2).copy_(x[1])
    assert torch.equal(nn.linear_packed((odd, scales), w, "MXFP8_E4M3"), y)
    zero = nn.linear_packed(torch.zeros(9, 64, device=DEV), w, "MXFP8_E4M3", out="MXFP8_E4M3")
    assert not zero[0].any() and not zero[1].any()


def test_lay_packed():
    from mxq import nn
    g = gen(23)
    x = random_pair((33, 160), "MXFP8_E4M3", g, DEV)
    for fmt in sorted(FORMATS):
        w = random_pair((50, 160), fmt, g, DEV)
        laid, name = nn.lay_packed(w, fmt)
        assert torch.equal(decode(laid, name), decode(w, fmt))
        assert torch.equal(nn.linear_packed(x, laid, name), nn.linear_packed(x, w, fmt))


def test_repeats():
    """The same bits on every run (K split over clusters, no atomics)."""
    from mxq import nn
    g = gen(29)
    for M in (1, 20, 64, 500):
        x, w = random_pair((M, 2048), "MXFP8_E4M3", g, DEV), random_pair((512, 2048), "MXFP8_E4M3", g, DEV)
        y = nn.linear_packed(x, w, "MXFP8_E4M3", out=torch.float32)
        for _ in range(3):
            assert torch.equal(nn.linear_packed(x, w, "MXFP8_E4M3", out=torch.float32), y)


@pytest.mark.parametrize("M", [8, 100, 600])
def test_chained_calls(M):
    """Calls that take one another's outputs, back to back: a product may be launched before the one before it has ended, and
    reads nothing until then. The same bits as with the device waited for after every call."""
    from mxq import nn
    g = gen(37 + M)
    x0 = torch.randn(M, 512, generator=g).to(DEV, torch.bfloat16)
    ws = [random_pair((512, 512), fmt, g, DEV) for fmt in ("MXFP8_E4M3", "MXFP4", "MXFP6_E3M2")]
    ws = [((c, s - 5), f) for (c, s), f in zip(ws, ("MXFP8_E4M3", "MXFP4", "MXFP6_E3M2"))]

    def chain(wait):
        x, seen = x0, []
        for i in range(24):
            w, fmt = ws[i % 3]
            packed = nn.linear_packed(x, w, fmt, activation="silu", out="MXFP8_E4M3")    # floats or the pair before
            if wait:
                torch.cuda.synchronize()
            x = nn.linear_packed(packed, w, fmt, residual=x0, out=torch.bfloat16) if i % 2 else packed
            if wait:
                torch.cuda.synchronize()
            seen.append(packed[0])
        return seen
    for a, b in zip(chain(False), chain(True)):
        assert torch.equal(a, b)


def test_laid_scales():
    """Scale rows that are laid out with their codes: odd numbers of blocks, the workspace's bytes and the scales of the
    next row all NaN's, one operand laid out or both, floats packed, rows of x in a plan's order."""
    from mxq import nn
    g = gen(31)
    for K in (8, 40, 1000, 2008, 2009):
        for M, N in ((1, 40), (70, 300), (600, 520)):
            for xf, wf in (("MXFP8_E4M3", "MXFP8_E5M2"), ("MXFP6_E3M2", "MXFP8_E4M3"), ("MXFP8_E4M3", "MXFP6_E2M3")):
                x, w = random_pair((M + 1, K), xf, g, DEV), random_pair((N + 1, K), wf, g, DEV)
                x[1][M:] = 255
                w[1][N:] = 255
                part = (x[0][:M], x[1][:M]), (w[0][:N], w[1][:N])
                torch.full((8 << 20,), 255, dtype=torch.uint8, device=DEV)               # what the allocator hands out next
                check(part[0], xf, part[1], wf, what=f"{M} x {N} x {K} {xf} {wf}")
            v = torch.randn(M, K, generator=g).to(DEV, torch.bfloat16)
            torch.full((8 << 20,), 255, dtype=torch.uint8, device=DEV)
            packed = nn.linear_packed(v, part[1], wf, x_fmt="MXFP8_E4M3", out=torch.float32)
            assert torch.isfinite(packed).all()
            aligned = torch.zeros(M, -(-K // 512) * 512, device=DEV, dtype=torch.bfloat16)     # the same values, nothing odd
            aligned[:, :K] = v
            wide = torch.zeros(N, aligned.shape[1], device=DEV, dtype=torch.uint8)
            wide[:, :K] = part[1][0]
            scales = torch.full((N, aligned.shape[1] // 32), 127, device=DEV, dtype=torch.uint8)
            scales[:, :part[1][1].shape[1]] = part[1][1]
            same = nn.linear_packed(aligned, (wide, scales), wf, x_fmt="MXFP8_E4M3", out=torch.float32)
            S = product64(v.double().abs(), decode(part[1], wf).abs())[0]
            # two sums of K values, the packed ones no more than twice the floats
            assert_close(packed, same.double(), 2 * (K + 1) * 2.0 ** -23 * 2 * S, torch.float32, f"floats {M} x {N} x {K}")
        for T in (6, 900):                               # few rows and many through a plan
            experts = torch.randint(0, 5, (T, 3), generator=g).int()
            x, w = random_pair((T, K), "MXFP8_E4M3", g, DEV), random_pair((5, 130, K), "MXFP6_E3M2", g, DEV)
            torch.full((8 << 20,), 255, dtype=torch.uint8, device=DEV)
            check_experts(x, "MXFP8_E4M3", w, "MXFP6_E3M2", experts, 5, True, what=f"plan {T} {K}")


def test_output_beyond_32_bits():
    """More than 2^31 values of y: the last rows and columns are where they belong."""
    from mxq import nn
    g = gen(31)
    M, N, K = 66000, 33024, 32
    x, w = random_pair((M, K), "MXFP8_E4M3", g, DEV), random_pair((N, K), "MXFP8_E4M3", g, DEV)
    y = nn.linear_packed(x, w, "MXFP8_E4M3", out=torch.bfloat16)
    for r in (slice(0, 40), slice(32500, 32540), slice(M - 40, M)):
        want, bound = product64(decode((x[0][r], x[1][r]), "MXFP8_E4M3"), decode(w, "MXFP8_E4M3"))
        assert_close(y[r], want, bound, torch.bfloat16, f"rows {r}")


# ----------------------------------------------------------------------------------------------- by expert
def plan_of(experts, E):
    from mxq import nn
    return nn.dispatch(experts.to(DEV), E)


def check_experts(x, xf, w, wf, experts, E, gather, bias=None, activation=None, out=torch.bfloat16, what=""):
    from mxq import nn
    plan = plan_of(experts, E)
    y = nn.experts_packed(x, w, wf, plan, gather=gather, x_fmt=xf, bias=bias, activation=activation, out=out)
    ends, order, k = plan.offsets.tolist(), plan.order.long(), experts.shape[1]
    rows = decode(x, xf)
    for e in range(E):
        a, b = ends[e], ends[e + 1]
        if a == b:
            continue
        mine = rows[order[a:b] // k] if gather else rows[a:b]
        want, bound = product64(mine, decode((w[0][e], w[1][e]), wf), None if bias is None else bias[e], activation)
        if isinstance(out, str):
            assert_packed((y[0][a:b], y[1][a:b]), want, bound, out, f"{what} expert {e}")
        else:
            assert_close(y[a:b], want, bound, out, f"{what} expert {e}")


PLANS = {
    "even": lambda T, E, k, g: torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]),
    "one": lambda T, E, k, g: torch.zeros(T, k, dtype=torch.long) + torch.arange(k),
    "last": lambda T, E, k, g: torch.full((T, k), E - 1),
    "holes": lambda T, E, k, g: torch.randint(-1, E, (T, k), generator=g),
    "none": lambda T, E, k, g: torch.full((T, k), -1),
}


@pytest.mark.parametrize("kind", sorted(PLANS))
@pytest.mark.parametrize("T,E,k", [(1, 4, 2), (7, 40, 3), (90, 5, 2), (700, 6, 4), (333, 64, 1)])
@pytest.mark.parametrize("gather", [True, False])
def test_plans(kind, T, E, k, gather):
    g = gen(T + E)
    experts = PLANS[kind](T, E, k, g).int()
    for K, N, act, out in ((160, 200, None, torch.bfloat16), (256, 384, "swiglu", "MXFP8_E4M3")):
        x = random_pair((T if gather else T * k, K), "MXFP8_E4M3", g, DEV)
        w = random_pair((E, N, K), "MXFP8_E4M3", g, DEV)
        bias = torch.randn(E, N, generator=g).to(DEV)
        check_experts(x, "MXFP8_E4M3", w, "MXFP8_E4M3", experts, E, gather, bias, act, out, f"{kind} {K}")


@pytest.mark.parametrize("T", [6, 800])
@pytest.mark.parametrize("wf", sorted(FORMATS))
@pytest.mark.parametrize("xf", ["MXFP8_E5M2", "MXFP4"])
def test_expert_formats(T, wf, xf):
    g = gen(37)
    experts = PLANS["holes"](T, 5, 2, g).int()
    for gather in (True, False):
        for K in (128, 96, 70):
            x = random_pair((T if gather else T * 2, K), xf, g, DEV)
            w = random_pair((5, 130, K), wf, g, DEV)
            check_experts(x, xf, w, wf, experts, 5, gather, None, "gelu", torch.float16, f"{xf} {wf} {K}")


def test_many_experts():
    g = gen(41)
    experts = torch.randint(0, 1024, (600, 4), generator=g).int()
    x, w = random_pair((600, 64), "MXFP8_E4M3", g, DEV), random_pair((1024, 40, 64), "MXFP8_E4M3", g, DEV)
    check_experts(x, "MXFP8_E4M3", w, "MXFP8_E4M3", experts, 1024, True)
    one = torch.zeros(2000, 1, dtype=torch.int32)
    w1 = (w[0][:1].contiguous(), w[1][:1].contiguous())
    x1 = random_pair((2000, 64), "MXFP8_E4M3", g, DEV)
    check_experts(x1, "MXFP8_E4M3", w1, "MXFP8_E4M3", one, 1, True)


def test_offsets_out_of_range_stay_in_bounds():
    """Offsets that no dispatch makes are cut to the rows that exist; the rows they leave alone keep what they had."""
    from mxq import nn
    g = gen(43)
    x, w = random_pair((10, 64), "MXFP8_E4M3", g, DEV), random_pair((3, 64, 64), "MXFP8_E4M3", g, DEV)
    order = torch.arange(10, dtype=torch.int32, device=DEV)
    for bad in ([-5, 4, 2000, 3000], [0, 20, 5, 12], [7, 3, 2, 1]):
        plan = nn.Dispatch(torch.tensor(bad, dtype=torch.int32, device=DEV), order, order.view(10, 1))
        nn.experts_packed(x, w, "MXFP8_E4M3", plan, gather=True)
    wild = nn.Dispatch(torch.tensor([0, 4, 8, 10], dtype=torch.int32, device=DEV), order * 1000 - 4000, order.view(10, 1))
    nn.experts_packed(x, w, "MXFP8_E4M3", wild, gather=True)
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    from mxq import nn
    g = gen(47)
    x, w = random_pair((4, 64), "MXFP8_E4M3", g, DEV), random_pair((6, 64), "MXFP8_E4M3", g, DEV)
    ok = dict(w=w, fmt="MXFP8_E4M3")
    cases = [
        ("uint8", lambda: nn.linear_packed(x, (w[0].int(), w[1]), "MXFP8_E4M3")),
        ("pair", lambda: nn.linear_packed(x, w[0], "MXFP8_E4M3")),
        ("shape", lambda: nn.linear_packed(x, (w[0], w[1][:, :1]), "MXFP8_E4M3")),
        ("2-D", lambda: nn.linear_packed(x, (w[0][0], w[1][0]), "MXFP8_E4M3")),
        ("values per row", lambda: nn.linear_packed(torch.zeros(4, 32, device=DEV), **ok)),
        ("element format", lambda: nn.linear_packed(x, w, "FP32")),
        ("Unknown format", lambda: nn.linear_packed(x, w, "FP7")),
        ("activation", lambda: nn.linear_packed(x, activation="tanh", **ok)),
        ("even number", lambda: nn.linear_packed(x, (w[0][:5], w[1][:5]), "MXFP8_E4M3", activation="swiglu")),
        ("bias", lambda: nn.linear_packed(x, bias=torch.zeros(5, device=DEV), **ok)),
        ("residual", lambda: nn.linear_packed(x, residual=torch.zeros(4, 6, device=DEV), **ok)),
        ("no residual", lambda: nn.linear_packed(x, residual=torch.zeros(4, 6, device=DEV, dtype=torch.bfloat16),
                                                 out="MXFP8_E4M3", **ok)),
        ("out must be", lambda: nn.linear_packed(x, out=torch.int32, **ok)),
        ("pairs up", lambda: nn.linear_packed(x, (w[0][:5], w[1][:5]), "MXFP8_E4M3", out="MXFP4")),
        ("float32, bfloat16", lambda: nn.linear_packed(torch.zeros(4, 64, device=DEV, dtype=torch.float64), **ok)),
        ("no values", lambda: nn.linear_packed(torch.zeros(4, 0, device=DEV), **ok)),
    ]
    e = torch.tensor([[0, 1]] * 4, dtype=torch.int32)
    plan = plan_of(e, 2)
    we = random_pair((2, 6, 64), "MXFP8_E4M3", g, DEV)
    cases += [
        ("3-D", lambda: nn.experts_packed(x, w, "MXFP8_E4M3", plan)),
        ("experts and w", lambda: nn.experts_packed(x, random_pair((3, 6, 64), "MXFP8_E4M3", g, DEV), "MXFP8_E4M3", plan)),
        ("no multiple", lambda: nn.experts_packed(random_pair((3, 64), "MXFP8_E4M3", g, DEV), we, "MXFP8_E4M3", plan)),
        ("rows and the plan", lambda: nn.experts_packed(x, we, "MXFP8_E4M3", plan, gather=False)),
        ("bias", lambda: nn.experts_packed(x, we, "MXFP8_E4M3", plan, bias=torch.zeros(6, device=DEV))),
        ("int32", lambda: nn.experts_packed(x, we, "MXFP8_E4M3", plan._replace(order=plan.order.long()))),
    ]
    for text, call in cases:
        with pytest.raises(ValueError, match=text):
            call()
