"""Plain 64-bit forms of the feed-forward operators on packed operands, for their tests: element codes by value tables,
scales as powers of two, products and activations in float64."""
import math

import torch

FORMATS = {"MXFP8_E4M3": (4, 3, 8, 448.0), "MXFP8_E5M2": (5, 2, 15, 57344.0), "MXFP6_E3M2": (3, 2, 4, 28.0),
           "MXFP6_E2M3": (2, 3, 2, 7.5), "MXFP4": (2, 1, 2, 6.0)}


def table(fmt):
    """Every code's value, float64."""
    e, m, _, _ = FORMATS[fmt]
    bias, out = 2 ** (e - 1) - 1, []
    for c in range(2 ** (1 + e + m)):
        sign, ex, man = -1.0 if c >> (e + m) else 1.0, (c >> m) % 2 ** e, c % 2 ** m
        v = man * 2.0 ** (1 - bias - m) if ex == 0 else (1 + man / 2 ** m) * 2.0 ** (ex - bias)
        if fmt == "MXFP8_E4M3" and (ex, man) == (15, 7):
            v = math.nan
        if fmt == "MXFP8_E5M2" and ex == 31:
            v = math.nan if man else math.inf
        out.append(sign * v)
    return torch.tensor(out, dtype=torch.float64)


def decode(pair, fmt):
    """The values of (codes, scales), float64, on their device."""
    codes, scales = pair
    if fmt == "MXFP4":
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    v = table(fmt).to(codes.device)[codes.long()]
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return v * s.repeat_interleave(32, -1)[..., :v.shape[-1]]


def random_pair(shape, fmt, g, device, spread=3):
    """Random finite codes and scales around 1."""
    *lead, K = shape
    e, m, _, _ = FORMATS[fmt]
    n = 2 ** (1 + e + m)
    codes = torch.randint(0, n, (*lead, K), generator=g, dtype=torch.int64)
    bad = ~torch.isfinite(table(fmt))[codes]
    codes[bad] = 1
    if fmt.startswith("MXFP8"):                       # a wide format's random codes would be all about its largest values
        low = torch.randint(0, 2 ** (m + 2), (*lead, K), generator=g) + (2 ** (e - 1) - 2 << m)
        codes = torch.where(codes % 3 == 0, codes, (codes & (n >> 1)) | low)
        codes[~torch.isfinite(table(fmt))[codes]] = 1
    codes = codes.to(torch.uint8)
    if fmt == "MXFP4":
        codes = codes[..., 0::2] | (codes[..., 1::2] << 4)
    scales = torch.randint(127 - spread, 128 + spread, (*lead, -(-K // 32)), generator=g).to(torch.uint8)
    return codes.contiguous().to(device), scales.to(device)


def act64(z, name):
    F = torch.nn.functional
    return {None: lambda t: t, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"),
            "silu": F.silu}[name](z)


#: the largest slope of each activation, rounded up
SLOPE = {None: 1.0, "relu": 1.0, "gelu": 1.13, "gelu_tanh": 1.13, "silu": 1.10}


def product64(x, w, bias=None, activation=None):
    """(y, bound): act(x w^T + bias) [* up] in float64 and how far a float32 evaluation may be from it.

    The products of the codes are exact. Each of the K additions may lose 2^-23 of the largest partial sum, itself at
    most S = sum |x w|: K 2^-23 S. The activation passes that on with its slope and adds its own error: a few ulp of its
    result and of its argument (2^-19 of each)."""
    K = x.shape[-1]
    z, S = x @ w.T, x.abs() @ w.abs().T
    dz = (K + 1) * 2.0 ** -23 * S
    if bias is not None:
        z = z + bias.double()
        dz = dz + 2.0 ** -23 * z.abs()
    gated = activation in ("swiglu", "geglu")
    name = {"swiglu": "silu", "geglu": "gelu"}.get(activation, activation)
    if gated:
        zg, zu = z.chunk(2, -1)
        dg, du = dz.chunk(2, -1)
    else:
        zg, dg = z, dz
    y = act64(zg, name)
    dy = SLOPE[name] * dg + (2.0 ** -19 * (y.abs() + zg.abs()) if name not in (None, "relu") else 0)
    if gated:
        dy = dy * (zu.abs() + du) + y.abs() * du + 2.0 ** -23 * (y * zu).abs()
        y = y * zu
    return y, dy


def rounding(y, dtype):
    """Half a step of dtype at y."""
    bits, low = {torch.float32: (24, -149), torch.bfloat16: (8, -133), torch.float16: (11, -24)}[dtype]
    return torch.maximum(y.abs() * 2.0 ** -bits, torch.full_like(y, 2.0 ** (low - 1)))


def assert_close(got, want, bound, dtype, what=""):
    """got (of dtype) within bound of want before its rounding."""
    tol = bound + rounding(want.abs() + bound, dtype) * (1 + 2.0 ** -8)
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    if dtype == torch.float16:                          # values from 65520 on round to Inf
        over = (want.abs() + bound >= 65520) & (got.double() == torch.sign(want) * math.inf)
        bad = torch.where(want.abs() - bound >= 65520, ~over, bad & ~over)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst {float((off / tol).nan_to_num(9e9).max()):.3g} of it"


def assert_packed(pair, want, bound, fmt, what=""):
    """(codes, scales) of fmt within half a step of want (+- bound), with the scales of the rule."""
    e, m, emax, top = FORMATS[fmt]
    K = want.shape[-1]
    pad = -K % 32
    blocks = torch.nn.functional.pad(want, (0, pad)).unflatten(-1, (-1, 32))
    room = torch.nn.functional.pad(bound, (0, pad)).unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1)
    slack = room.amax(-1)

    def byte(a):
        ex = torch.frexp(a)[1] - 1 - emax + 127
        return torch.where(a > 0, ex, torch.zeros_like(ex)).clamp(0, 254)
    lo, hi = byte((amax - slack).clamp_min(0)), byte(amax + slack)
    got = pair[1].long()
    assert ((got >= lo) & (got <= hi)).all(), f"{what}: scales"
    X = torch.exp2(got.double() - 127).repeat_interleave(32, -1)[..., :K]
    z = (want / X).clamp(-top, top)
    low = 2.0 ** (2 - 2 ** (e - 1))                      # the smallest normal value
    step = torch.exp2(torch.floor(torch.log2((z.abs() + bound / X).clamp_min(low))) - m) * X
    off = (decode(pair, fmt) - z * X).abs()
    tol = 0.5 * step * (1 + 2.0 ** -10) + bound * (1 + 2.0 ** -10)
    assert (off <= tol).all(), f"{what}: codes, {int((off > tol).sum())} off, worst {float((off / tol).max()):.3g}"


# ----------------------------------------------------------------------------------------------- routing
def route64(logits, k, score, bias=None, groups=1, keep=1, top2=False, renormalize=False, scale=1.0):
    """(weights, experts) row by row in float64; the margin between any two compared choice values that differ."""
    T, E = logits.shape
    W, X, margin = torch.zeros(T, k, dtype=torch.float64), torch.full((T, k), -1, dtype=torch.int32), math.inf
    for t in range(T):
        l = logits[t].double()
        bad = bool(l.isnan().any())
        live = [e for e in range(E) if l[e] > -math.inf]
        alive = set(live)
        if score == "softmax":
            top = max([float(l[e]) for e in live], default=0.0)
            ex = torch.tensor([math.exp(float(l[e]) - top) if e in alive else 0.0 for e in range(E)], dtype=torch.float64)
            s = ex / ex.sum() if live else ex
        else:
            s = torch.tensor([float(torch.sigmoid(l[e])) if e in alive else 0.0 for e in range(E)], dtype=torch.float64)
        c = {e: float(l[e]) if bias is None else float(s[e]) + float(bias[e]) for e in live}
        if groups > 1:
            run, value = E // groups, {}
            for gr in range(groups):
                mine = sorted((c[e] for e in live if e // run == gr), reverse=True)
                if mine:
                    value[gr] = sum(mine[:2]) if top2 else mine[0]
            kept = sorted(value, key=lambda gr: (-value[gr], gr))[:keep]
            vs = sorted(value.values())
            margin = min([margin] + [b - a for a, b in zip(vs, vs[1:]) if b > a])
            c = {e: v for e, v in c.items() if e // run in kept}
        vs = sorted(c.values())
        margin = min([margin] + [b - a for a, b in zip(vs, vs[1:]) if b > a])
        chosen = sorted(c, key=lambda e: (-c[e], e))[:k]
        w = s[chosen]
        if renormalize:
            w = w / (w.sum() + 1e-20)
        W[t, :len(chosen)] = w * scale
        X[t, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
        if bad:
            W[t] = math.nan
    return W, X, margin


def route_backward64(grad, logits, experts, score, renormalize, scale):
    x = logits.detach().double().clone().requires_grad_(True)
    with torch.enable_grad():
        s = torch.softmax(x, -1) if score == "softmax" else torch.sigmoid(x)
        live = experts >= 0
        w = torch.where(live, s.gather(1, experts.long().clamp_min(0)), torch.zeros((), dtype=torch.float64, device=x.device))
        if renormalize:
            w = w / (w.sum(1, keepdim=True) + 1e-20)
        (w * scale * torch.where(live, grad.double(), torch.zeros_like(w))).sum().backward()
    return x.grad


def dispatch64(experts, E):
    """(offsets, order, where) by a stable sort on the host."""
    flat = experts.flatten().tolist()
    slots = sorted((i for i, e in enumerate(flat) if 0 <= e < E), key=lambda i: flat[i])
    offsets = [0] * (E + 1)
    for i in slots:
        offsets[flat[i] + 1] += 1
    for e in range(E):
        offsets[e + 1] += offsets[e]
    where = [-1] * len(flat)
    for p, i in enumerate(slots):
        where[i] = p
    order = slots + [-1] * (len(flat) - len(slots))
    as_t = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return as_t(offsets), as_t(order), as_t(where).view(experts.shape)
