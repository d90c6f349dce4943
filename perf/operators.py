"""The measured cases of the feed-forward operators on packed MX operands: the router (nn.route and nn.dispatch, and
the router's gradient), the product with its epilogue (nn.linear_packed), the experts' products (nn.experts_packed) and
the weighted sum of the experts' outputs (nn.combine, and its gradients).

Each operator in its plain form (`own` false: elementary torch operations in 32 bits) and as the package's call (`own`
true). Operands are what a serving or tuning program holds: uint8 OCP codes with one E8M0 scale byte per 32 values
along the last dimension (FP4: two codes per byte, the even one low).
"""
import math
import sys

import torch

own = False

DEV = "cuda"
BLOCK = 32
EPS = 1e-20                                    # added to the sum that renormalises the routing weights

#: element formats: exponent bits, mantissa bits, exponent of the largest value, the largest value
FORMATS = {"MXFP8_E4M3": (4, 3, 8, 448.0), "MXFP8_E5M2": (5, 2, 15, 57344.0), "MXFP6_E3M2": (3, 2, 4, 28.0),
           "MXFP6_E2M3": (2, 3, 2, 7.5), "MXFP4": (2, 1, 2, 6.0)}
FLOATS = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GATED = ("swiglu", "geglu")


def _nn():
    if "microscaling-quant_b200" not in sys.path:
        sys.path.insert(0, "microscaling-quant_b200")
    from mxq import nn
    return nn


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the router of one decoding batch: sigmoid scores with a balance bias, 8 groups of which 4 are kept
        {"name": "route decode", "op": "route", "T": 16, "E": 128, "k": 8, "score": "sigmoid", "bias": True, "groups": 8,
         "keep": 4, "renormalize": True, "dtype": "bf16"},
        # the router of a long prompt
        {"name": "route prompt", "op": "route", "T": 8192, "E": 256, "k": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "keep": 4, "renormalize": True, "dtype": "f32"},
        # the router's gradient over a training batch, softmax scores
        {"name": "route gradient", "op": "route_grad", "T": 8191, "E": 64, "k": 6, "score": "softmax",
         "renormalize": True, "dtype": "bf16"},
        # one token through the gated up-projection of a 2048-wide model
        {"name": "linear one token", "op": "linear", "M": 1, "N": 8192, "K": 2048, "x": "packed", "x_fmt": "MXFP8_E4M3",
         "fmt": "MXFP8_E4M3", "bias": False, "activation": "swiglu", "residual": False, "out": "bf16"},
        # a decoding batch through the down-projection, 4-bit weights, the activations packed within the call
        {"name": "linear decode", "op": "linear", "M": 24, "N": 4096, "K": 8192, "x": "bf16", "x_fmt": "MXFP8_E4M3",
         "fmt": "MXFP4", "bias": False, "activation": "none", "residual": True, "out": "bf16"},
        # ragged sizes: K is no multiple of the block, rows end inside every tile, 6-bit weights
        {"name": "linear ragged", "op": "linear", "M": 777, "N": 1000, "K": 2008, "x": "packed", "x_fmt": "MXFP8_E5M2",
         "fmt": "MXFP6_E3M2", "bias": True, "activation": "gelu", "residual": True, "out": "f16"},
        # a prompt through an up-projection whose output the next product takes packed
        {"name": "linear prompt", "op": "linear", "M": 4096, "N": 8192, "K": 2048, "x": "packed", "x_fmt": "MXFP8_E4M3",
         "fmt": "MXFP8_E4M3", "bias": False, "activation": "swiglu", "residual": False, "out": "MXFP8_E4M3"},
        # the largest: a square layer over 8192 tokens with bias, activation and residual
        {"name": "linear large", "op": "linear", "M": 8192, "N": 8192, "K": 8192, "x": "packed", "x_fmt": "MXFP8_E4M3",
         "fmt": "MXFP8_E4M3", "bias": True, "activation": "silu", "residual": True, "out": "bf16"},
        # a decoding batch through the experts' gated up-projections
        {"name": "experts decode", "op": "experts", "T": 8, "E": 64, "k": 6, "N": 2048, "K": 2048, "gather": True,
         "x_fmt": "MXFP8_E4M3", "fmt": "MXFP8_E4M3", "bias": False, "activation": "swiglu", "out": "MXFP8_E4M3"},
        # a prompt through the experts' down-projections, rows already in the experts' order
        {"name": "experts prompt", "op": "experts", "T": 4096, "E": 64, "k": 6, "N": 2048, "K": 1024, "gather": False,
         "x_fmt": "MXFP8_E4M3", "fmt": "MXFP8_E4M3", "bias": True, "activation": "none", "out": "bf16"},
        # the weighted sum for a decoding batch
        {"name": "combine decode", "op": "combine", "T": 24, "k": 6, "E": 64, "N": 2048, "residual": True, "dtype": "bf16"},
        # its gradients over a training batch
        {"name": "combine gradient", "op": "combine_grad", "T": 4096, "k": 6, "E": 64, "N": 2048, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "route_grad", "linear", "linear", "linear", "experts", "experts", "combine", "combine_grad"])
    if op in ("route", "route_grad"):
        E = rng.choice([8, 16, 40, 64, 96, 128, 160, 256])
        score = rng.choice(["softmax", "sigmoid"])
        c = {"op": op, "T": _log(rng, 1, 8192), "E": E, "k": rng.randint(1, 8), "score": score,
             "renormalize": rng.random() < 0.6, "dtype": rng.choice(["bf16", "f16", "f32"])}
        if op == "route":
            grouped = rng.random() < 0.5
            c |= {"bias": score == "sigmoid" and rng.random() < 0.7, "groups": 4 if grouped else 1,
                  "keep": 2 if grouped else 1}
            c["k"] = min(c["k"], E // 2) if grouped else c["k"]
        return c
    if op == "linear":
        M, N, K = _log(rng, 1, 8192), 2 * _log(rng, 32, 4096), 2 * _log(rng, 32, 4096)
        if rng.random() < 0.6:
            K = -(-K // 128) * 128
        act = rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh", "swiglu", "geglu"])
        out = rng.choice(["bf16", "bf16", "f16", "f32", "MXFP8_E4M3"])
        return {"op": op, "M": M, "N": N, "K": K, "x": rng.choice(["packed", "packed", "bf16", "f32"]),
                "x_fmt": rng.choice(["MXFP8_E4M3", "MXFP8_E4M3", "MXFP8_E5M2"]), "fmt": rng.choice(sorted(FORMATS)),
                "bias": rng.random() < 0.5, "activation": act, "residual": out in FLOATS and rng.random() < 0.5,
                "out": out}
    if op == "experts":
        E = rng.choice([4, 8, 16, 32, 64])
        return {"op": op, "T": _log(rng, 1, 4096), "E": E, "k": rng.randint(1, min(6, E)), "N": 2 * _log(rng, 64, 1024),
                "K": 32 * _log(rng, 4, 64), "gather": rng.random() < 0.5, "x_fmt": "MXFP8_E4M3",
                "fmt": rng.choice(["MXFP8_E4M3", "MXFP8_E4M3", "MXFP4"]), "bias": rng.random() < 0.5,
                "activation": rng.choice(["none", "gelu", "swiglu", "swiglu"]),
                "out": rng.choice(["bf16", "f16", "MXFP8_E4M3"])}
    E = rng.choice([8, 32, 64])
    return {"op": op, "T": _log(rng, 1, 4096), "k": rng.randint(1, 8), "E": E, "N": _log(rng, 64, 4096),
            **({"residual": rng.random() < 0.5} if op == "combine" else {}), "dtype": rng.choice(["bf16", "f16", "f32"])}


# ----------------------------------------------------------------------------------- packed operands
def _table(fmt):
    """The values of a format's codes, as a float32 tensor."""
    e, m, _, _ = FORMATS[fmt]
    bias, vals = 2 ** (e - 1) - 1, []
    for c in range(2 ** (1 + e + m)):
        ex, man = (c >> m) % 2 ** e, c % 2 ** m
        v = man * 2.0 ** (1 - bias - m) if ex == 0 else (1 + man / 2 ** m) * 2.0 ** (ex - bias)
        if fmt == "MXFP8_E4M3" and ex == 15 and man == 7:
            v = float("nan")
        if fmt == "MXFP8_E5M2" and ex == 31:
            v = float("nan") if man else float("inf")
        vals.append(-v if c >> (e + m) else v)
    return torch.tensor(vals, dtype=torch.float32, device=DEV)


def _scale_exponent(amax, emax):
    """floor(log2 amax) - emax within what an E8M0 byte holds; the lowest exponent for a block of zeros."""
    ex = torch.frexp(amax)[1] - 1 - emax
    return torch.where(amax > 0, ex, torch.full_like(ex, -127)).clamp(-127, 127)


def _blocks(v):
    """(..., K) padded with zeros to (..., blocks, 32)."""
    pad = -v.shape[-1] % BLOCK
    if pad:
        v = torch.nn.functional.pad(v, (0, pad))
    return v.unflatten(-1, (-1, BLOCK))


def _encode8(v, fmt):
    """The 8-bit codes (as float8 values) and scale exponents of v (float32 or float64), round to nearest even."""
    _, _, emax, top = FORMATS[fmt]
    b = _blocks(v)
    ex = _scale_exponent(b.abs().amax(-1), emax)
    z = torch.ldexp(b, -ex[..., None]).clamp(-top, top)
    q = z.float().to(torch.float8_e4m3fn if fmt == "MXFP8_E4M3" else torch.float8_e5m2)
    return q.flatten(-2)[..., :v.shape[-1]], ex


def _pack(v, fmt):
    """(codes, scales) of v in the packed form, for making inputs."""
    if fmt.startswith("MXFP8"):
        q, ex = _encode8(v, fmt)
        return q.contiguous().view(torch.uint8), (ex + 127).to(torch.uint8)
    e, m, emax, top = FORMATS[fmt]
    half = _table(fmt)[:2 ** (e + m)]
    b = _blocks(v)
    ex = _scale_exponent(b.abs().amax(-1), emax)
    z = torch.ldexp(b, -ex[..., None]).flatten(-2)[..., :v.shape[-1]]
    codes = torch.bucketize(z.abs().contiguous(), (half[1:] + half[:-1]) / 2).to(torch.uint8)
    codes |= (z < 0).to(torch.uint8) << (e + m)
    if fmt == "MXFP4":
        codes = codes[..., 0::2] | (codes[..., 1::2] << 4)
    return codes.contiguous(), (ex + 127).to(torch.uint8)


def _values(codes, scales, fmt, dtype=torch.float32):
    """The values a packed operand stands for."""
    if fmt == "MXFP4":
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    if fmt == "MXFP8_E4M3":
        v = codes.view(torch.float8_e4m3fn).to(dtype)
    elif fmt == "MXFP8_E5M2":
        v = codes.view(torch.float8_e5m2).to(dtype)
    else:
        v = _table(fmt).to(dtype)[codes.int()]
    one = torch.ones((), dtype=dtype, device=codes.device)
    s = torch.ldexp(one, scales.int() - 127)
    return v * s.repeat_interleave(BLOCK, -1)[..., :v.shape[-1]]


# -------------------------------------------------------------------------------------------- inputs
def _experts_of(T, E, k, g):
    """k different experts per token from skewed random preferences, as a trained router gives them."""
    pref = torch.randn(T, E, device=DEV, generator=g) + 0.7 * torch.randn(E, device=DEV, generator=g)
    return torch.topk(pref, k, dim=-1).indices.to(torch.int32)


def _plan(experts, E):
    """The experts' order of the slots: where each expert's rows begin, the slot at each place, the place of each slot."""
    flat = experts.flatten().long()
    order = torch.argsort(flat, stable=True)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
    offsets[1:] = torch.cumsum(torch.bincount(flat, minlength=E), 0)
    where = torch.empty_like(order)
    where[order] = torch.arange(order.numel(), device=DEV)
    return offsets, order.to(torch.int32), where.to(torch.int32).view(experts.shape)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c, s = case, {"case": case}

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    if c["op"] in ("route", "route_grad"):
        s["logits"] = (2.0 * randn(c["T"], c["E"])).to(FLOATS[c["dtype"]])
        s["bias"] = 0.05 * randn(c["E"]) if c.get("bias") else None
        if c["op"] == "route_grad":
            s["grad"] = randn(c["T"], c["k"])
            s["experts"] = torch.sort(s["logits"], dim=-1, descending=True, stable=True).indices[:, :c["k"]].to(torch.int32)
        return s
    if c["op"] == "linear":
        x = randn(c["M"], c["K"]) * (1 + 4 * (torch.rand(c["K"], device=DEV, generator=g) < 0.01))
        s["x"] = _pack(x, c["x_fmt"]) if c["x"] == "packed" else x.to(FLOATS[c["x"]])
        s["w"] = _pack(randn(c["N"], c["K"]) / math.sqrt(c["K"]), c["fmt"])
        s["bias"] = 0.1 * randn(c["N"]) if c["bias"] else None
        s["residual"] = randn(c["M"], _width(c)).to(FLOATS[c["out"]]) if c["residual"] else None
        return s
    experts = _experts_of(c["T"], c["E"], c["k"], g)
    s["offsets"], s["order"], s["where"] = _plan(experts, c["E"])
    if c["op"] == "experts":
        s["experts"] = experts
        counts = torch.bincount(experts.flatten().long(), minlength=c["E"])
        s["live"] = torch.nonzero(counts).flatten()           # the experts that have rows, and the longest's rows
        s["most"] = int(counts.max())
        s["x"] = _pack(randn(c["T"] if c["gather"] else c["T"] * c["k"], c["K"]), c["x_fmt"])
        parts = [_pack(randn(c["N"], c["K"]) / math.sqrt(c["K"]), c["fmt"]) for _ in range(c["E"])]
        s["w"] = tuple(torch.stack(p) for p in zip(*parts))
        s["bias"] = 0.1 * randn(c["E"], c["N"]) if c["bias"] else None
        return s
    dt = FLOATS[c["dtype"]]
    s["z"] = randn(c["T"] * c["k"], c["N"]).to(dt)
    s["weights"] = torch.softmax(randn(c["T"], c["k"]), -1)
    if c["op"] == "combine":
        s["residual"] = randn(c["T"], c["N"]).to(dt) if c["residual"] else None
    else:
        s["grad"] = randn(c["T"], c["N"]).to(dt)
    return s


def _width(c):
    return c["N"] // 2 if c["activation"] in GATED else c["N"]


# ------------------------------------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    c, nn = s["case"], _nn()
    if c["op"] == "route":
        weights, experts = nn.route(s["logits"], c["k"], score=c["score"], bias=s["bias"], groups=c["groups"],
                                    keep=c["keep"], group_score="top2" if c["bias"] else "max",
                                    renormalize=c["renormalize"], scale=2.5)
        plan = nn.dispatch(experts, c["E"])
        return weights, experts, plan.offsets, plan.order, plan.where
    if c["op"] == "route_grad":
        return nn.route_backward(s["grad"], s["logits"], s["experts"], score=c["score"], renormalize=c["renormalize"],
                                 scale=2.5)
    act = None if c.get("activation") == "none" else c.get("activation")
    out = FLOATS.get(c.get("out"), c.get("out"))
    if c["op"] == "linear":
        y = nn.linear_packed(s["x"], s["w"], c["fmt"], x_fmt=c["x_fmt"], bias=s["bias"], activation=act,
                             residual=s["residual"], out=out)
    elif c["op"] == "experts":
        y = nn.experts_packed(s["x"], s["w"], c["fmt"], nn.Dispatch(s["offsets"], s["order"], s["where"]),
                              gather=c["gather"], x_fmt=c["x_fmt"], bias=s["bias"], activation=act, out=out)
    elif c["op"] == "combine":
        return nn.combine(s["z"], s["weights"], nn.Dispatch(s["offsets"], s["order"], s["where"]), residual=s["residual"])
    else:
        return nn.combine_backward(s["grad"], s["z"], s["weights"], nn.Dispatch(s["offsets"], s["order"], s["where"]))
    if isinstance(y, tuple):
        return y[0].view(torch.float8_e4m3fn), y[1].view(torch.float8_e8m0fnu)
    return y


def _scores(logits, score):
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-logits))
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _activate(acc, act):
    if act in GATED:
        gate, up = acc.chunk(2, -1)
        return _activate(gate, "silu" if act == "swiglu" else "gelu") * up
    if act == "relu":
        return torch.clamp_min(acc, 0)
    if act == "silu":
        return acc / (1 + torch.exp(-acc))
    if act == "gelu":
        return 0.5 * acc * (1 + torch.erf(acc * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * acc * (1 + torch.tanh(math.sqrt(2 / math.pi) * (acc + 0.044715 * acc * acc * acc)))
    return acc


def _emit(y, out):
    if out in FLOATS:
        return y.to(FLOATS[out])
    q, ex = _encode8(y, out)
    return q, (ex + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _first(choice, k):
    """The k largest of each row, ties to the lowest index."""
    return torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, :k]


def _run_plain(s):
    c = s["case"]
    if c["op"] == "route":
        l = s["logits"].float()
        scores = _scores(l, c["score"])
        choice = l if s["bias"] is None else scores + s["bias"]
        if c["groups"] > 1:
            by = choice.unflatten(-1, (c["groups"], -1))
            best = torch.topk(by, 2, -1).values.sum(-1) if c["bias"] else by.amax(-1)
            kept = torch.zeros_like(best, dtype=torch.bool).scatter_(-1, _first(best, c["keep"]), True)
            choice = torch.where(kept[..., None], by, float("-inf")).flatten(-2)
        experts = _first(choice, c["k"])
        weights = scores.gather(-1, experts)
        if c["renormalize"]:
            weights = weights / (weights.sum(-1, keepdim=True) + EPS)
        return (weights * 2.5, experts.to(torch.int32), *_plan(experts, c["E"]))
    if c["op"] == "route_grad":
        l, idx = s["logits"].float(), s["experts"].long()
        scores = _scores(l, c["score"])
        picked, grad = scores.gather(-1, idx), s["grad"] * 2.5
        if c["renormalize"]:
            total = picked.sum(-1, keepdim=True) + EPS
            grad = (grad - (grad * picked).sum(-1, keepdim=True) / total) / total
        full = torch.zeros_like(scores).scatter_(-1, idx, grad)
        if c["score"] == "sigmoid":
            return (full * scores * (1 - scores)).to(s["logits"].dtype)
        return (scores * (full - (full * scores).sum(-1, keepdim=True))).to(s["logits"].dtype)
    if c["op"] == "linear":
        x = s["x"]
        if c["x"] != "packed":
            q, ex = _encode8(x.float(), c["x_fmt"])
            x = q.contiguous().view(torch.uint8), (ex + 127).to(torch.uint8)
        acc = _values(*x, c["x_fmt"]) @ _values(*s["w"], c["fmt"]).T
        if s["bias"] is not None:
            acc = acc + s["bias"]
        y = _activate(acc, c["activation"])
        return _emit(y if s["residual"] is None else y + s["residual"].float(), c["out"])
    if c["op"] == "experts":
        live, first = s["live"], s["offsets"][:-1].long()
        x = _values(*s["x"], c["x_fmt"])
        x = x[s["order"].long() // c["k"]] if c["gather"] else x
        expert = s["experts"].flatten().long()[s["order"].long()]         # of each row, in the experts' order
        row = torch.arange(expert.numel(), device=DEV) - first[expert]
        at = torch.searchsorted(live, expert)
        padded = x.new_zeros(live.numel(), s["most"], c["K"])
        padded[at, row] = x
        w = _values(s["w"][0][live], s["w"][1][live], c["fmt"])
        acc = torch.bmm(padded, w.transpose(1, 2))[at, row]
        if s["bias"] is not None:
            acc = acc + s["bias"][expert]
        return _emit(_activate(acc, c["activation"]), c["out"])
    rows = s["z"][s["where"].long()].float()                               # T x k x N
    if c["op"] == "combine":
        y = (rows * s["weights"][..., None]).sum(1)
        return (y if s["residual"] is None else y + s["residual"].float()).to(s["z"].dtype)
    dy = s["grad"].float()
    dw = (rows * dy[:, None]).sum(-1)
    order = s["order"].long()
    dz = s["weights"].flatten()[order][:, None] * dy[order // c["k"]]
    return dz.to(s["z"].dtype), dw


# ------------------------------------------------------------------------------------------- the floor
def work(case):
    c = case
    if c["op"] in ("route", "route_grad"):
        size = 4 if c["dtype"] == "f32" else 2
        slots = c["T"] * c["k"]
        if c["op"] == "route":
            return {"bytes": c["T"] * c["E"] * size + slots * 16 + 4 * c["E"], "flops": 4 * c["T"] * c["E"]}
        return {"bytes": 2 * c["T"] * c["E"] * size + slots * 8, "flops": 6 * c["T"] * c["E"]}
    if c["op"] in ("linear", "experts"):
        bits = 0.5 if c["fmt"] == "MXFP4" else 1
        wrow = c["K"] * bits + c["K"] / BLOCK
        xrow = c["K"] * (1 + 1 / BLOCK)
        orow = _width(c) * {"bf16": 2, "f16": 2, "f32": 4}.get(c["out"], 1 + 1 / BLOCK)
        if c["op"] == "linear":
            xrow = {"bf16": 2.0, "f32": 4.0}.get(c["x"], 1 + 1 / BLOCK) * c["K"]
            moved = c["M"] * (xrow + orow * (2 if c["residual"] else 1)) + c["N"] * (wrow + (4 if c["bias"] else 0))
            return {"bytes": moved, "flops": 2 * c["M"] * c["N"] * c["K"]}
        slots = c["T"] * c["k"]
        live = min(c["E"], slots)
        moved = (c["T"] if c["gather"] else slots) * xrow + slots * orow + live * c["N"] * (wrow + (4 if c["bias"] else 0))
        return {"bytes": moved, "flops": 2 * slots * c["N"] * c["K"]}
    size = 4 if c["dtype"] == "f32" else 2
    slots = c["T"] * c["k"]
    if c["op"] == "combine":
        return {"bytes": size * c["N"] * (slots + c["T"] * (2 if c["residual"] else 1)) + slots * 8,
                "flops": 2 * slots * c["N"]}
    return {"bytes": size * c["N"] * (2 * slots + c["T"]) + slots * 16, "flops": 3 * slots * c["N"]}


# ------------------------------------------------------------------------------------ in 64 bits, apart
def exact(case, seed):
    """run's outputs from the definition in float64 (the experts and their order, which are whole numbers, are None)."""
    c, s = case, prepare(case, seed)
    f8 = torch.float64
    if c["op"] in ("route", "route_grad"):
        l = s["logits"].to(f8)
        p = torch.sigmoid(l) if c["score"] == "sigmoid" else torch.softmax(l, -1)
        if c["op"] == "route":
            pick = (l if s["bias"] is None else p + s["bias"].to(f8)).clone()
            T, G = c["T"], c["groups"]
            if G > 1:
                v = pick.view(T, G, -1)
                top = v.sort(-1).values
                g = top[..., -1] + top[..., -2] if c["bias"] else top[..., -1]
                drop = g.sort(dim=-1, descending=True, stable=True).indices[:, c["keep"]:]
                v[torch.arange(T, device=DEV)[:, None], drop] = float("-inf")
            idx = pick.sort(dim=-1, descending=True, stable=True).indices[:, :c["k"]]
            w = torch.take_along_dim(p, idx, 1)
            if c["renormalize"]:
                w = w / (w.sum(1, keepdim=True) + EPS)
            return w * 2.5, None, None, None, None
        p.requires_grad_(False)
        x = l.clone().requires_grad_(True)
        with torch.enable_grad():
            q = torch.sigmoid(x) if c["score"] == "sigmoid" else torch.softmax(x, -1)
            w = torch.take_along_dim(q, s["experts"].long(), 1)
            if c["renormalize"]:
                w = w / (w.sum(1, keepdim=True) + EPS)
            (w * 2.5 * s["grad"].to(f8)).sum().backward()
        return x.grad

    def decoded(codes, scales, fmt):
        e, m, _, _ = FORMATS[fmt]
        b = codes.to(torch.int64)
        if fmt == "MXFP4":
            b = torch.stack((b % 16, b // 16), -1).reshape(*b.shape[:-1], -1)
        man, ex, neg = b % 2 ** m, b // 2 ** m % 2 ** e, b // 2 ** (m + e)
        mag = torch.where(ex == 0, man.to(f8) * 2.0 ** (2 - 2 ** (e - 1) - m),
                          (2 ** m + man).to(f8) * torch.exp2((ex - 2 ** (e - 1) + 1 - m).to(f8)))
        mag = torch.where(neg == 1, -mag, mag)
        return mag * torch.exp2(scales.to(f8) - 127).repeat_interleave(32, -1)[..., :mag.shape[-1]]

    def act(a, name):
        F = torch.nn.functional
        if name in GATED:
            h = a.shape[-1] // 2
            return (F.silu if name == "swiglu" else F.gelu)(a[..., :h]) * a[..., h:]
        return {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu,
                "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[name](a)

    def given(y):
        if c["out"] in FLOATS:
            return y
        pad = -y.shape[-1] % 32
        b = torch.nn.functional.pad(y, (0, pad)).view(y.shape[0], -1, 32)
        ex = (torch.floor(torch.log2(b.abs().amax(-1))) - 8).clamp(-127, 127)       # of the 4-bit-exponent 8-bit format
        z = b * torch.exp2(-ex)[..., None]
        step = torch.exp2(torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6))) - 3)
        z = (torch.round(z / step) * step).clamp(-448, 448)
        return z.reshape(y.shape[0], -1)[:, :y.shape[1]], torch.exp2(ex)

    if c["op"] == "linear":
        if c["x"] == "packed":
            x = decoded(*s["x"], c["x_fmt"])
        else:
            _, m, emax, top = FORMATS[c["x_fmt"]]
            low = 2.0 ** (-6 if c["x_fmt"] == "MXFP8_E4M3" else -14)
            v = s["x"].to(f8)
            b = torch.nn.functional.pad(v, (0, -v.shape[1] % 32)).view(v.shape[0], -1, 32)
            ex = (torch.floor(torch.log2(b.abs().amax(-1))) - emax).clamp(-127, 127)[..., None]
            z = b * torch.exp2(-ex)
            step = torch.exp2(torch.floor(torch.log2(z.abs().clamp_min(low))) - m)
            x = ((torch.round(z / step) * step).clamp(-top, top) * torch.exp2(ex)).view(v.shape[0], -1)[:, :v.shape[1]]
        y = x @ decoded(*s["w"], c["fmt"]).T
        if s["bias"] is not None:
            y += s["bias"].to(f8)
        y = act(y, c["activation"])
        return given(y if s["residual"] is None else y + s["residual"].to(f8))
    if c["op"] == "experts":
        x = decoded(*s["x"], c["x_fmt"])
        if c["gather"]:
            x = x.index_select(0, s["order"].long() // c["k"])
        ends, parts = s["offsets"].tolist(), []
        for e in range(c["E"]):
            if ends[e] == ends[e + 1]:
                continue
            y = x[ends[e]:ends[e + 1]] @ decoded(s["w"][0][e], s["w"][1][e], c["fmt"]).T
            parts.append(y if s["bias"] is None else y + s["bias"][e].to(f8))
        return given(act(torch.cat(parts), c["activation"]))
    z, w = s["z"].to(f8), s["weights"].to(f8)
    at = s["where"].long()
    if c["op"] == "combine":
        y = torch.einsum("tk,tkn->tn", w, z[at])
        return y if s["residual"] is None else y + s["residual"].to(f8)
    dy = s["grad"].to(f8)
    dz = torch.empty_like(z)
    dz[at.flatten()] = (w[..., None] * dy[:, None]).reshape(-1, c["N"])
    return dz, torch.einsum("tn,tkn->tk", dy, z[at])
