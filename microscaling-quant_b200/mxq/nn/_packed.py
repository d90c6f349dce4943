"""Products of packed MX operands on the tensor cores, dense and by expert (no reference counterpart). Inference only: of their
arguments the residual alone has a gradient (the result's); one that reaches a float x or a bias raises in backward.

    y = linear_packed(x, w, "MXFP8_E4M3", bias=b, activation="silu", residual=r)       ... x K, N x K -> ... x F
    z = experts_packed(x, w, "MXFP8_E4M3", plan, activation="swiglu", out="MXFP8_E4M3")

An operand is a pair (codes, scales) as block.ocp.quantize_packed(V, fmt, axis=-1) gives it: uint8 codes (FP4 two per
byte) and one E8M0 byte per 32 values of the last dimension. x may also be a float tensor: its rows are then packed to
`x_fmt` within the call, by the rule of a packed output.

    acc = sum_k x[.., k] w[n, k]            the values the codes stand for; products exact, sums float32
    y   = act(acc + bias) [* up] + residual

Activations: None, "relu", "gelu" (erf), "gelu_tanh", "silu", and the gated "swiglu" / "geglu", whose first N / 2 rows of
w are the gate's and the others the up projection's (F = N / 2; else F = N). `out` is a float dtype or a format name; a
packed output is a pair again: the scale 2^(floor(log2 amax) - emax) per 32 columns, codes rounded to nearest even and
saturated, the scale of a block that holds an Inf or a NaN 0xFF (NaN).

8-bit codes whose rows are multiples of 16 bytes, and FP4 codes with K a multiple of 128, are read as they are. Other
codes (FP6, ragged or unaligned rows) are laid out as 8-bit codes first, in every call; `lay_packed` does it once for
weights that are kept.
"""
from typing import NamedTuple, Optional, Tuple, Union

import ctypes

import torch

from .. import _lib
from ..block import BLOCK
from ..element_quant.formats import FORMATS, Format, get

__all__ = ["ACTIVATIONS", "Dispatch", "linear_packed", "experts_packed", "lay_packed"]

ACTIVATIONS = (None, "relu", "gelu", "gelu_tanh", "silu", "swiglu", "geglu")
GATED = ("swiglu", "geglu")
FIRST_GATED = 5
FLOATS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
PACKED = 3

Pair = Tuple[torch.Tensor, torch.Tensor]


class Dispatch(NamedTuple):
    """The slots (token-major, T x k flattened) in the order of their experts, as nn.dispatch makes it (int32)."""
    offsets: torch.Tensor   # (experts + 1): where each expert's places begin
    order: torch.Tensor     # (slots): the slot at each place, -1 at the places beyond offsets[-1]
    where: torch.Tensor     # (T, k): the place of each slot, -1 for a slot left out


def _format(fmt, who: str) -> Format:
    f = FORMATS.get(fmt) if type(fmt) is str else None
    if f is None:
        f = get(fmt)
        if f is None:
            raise ValueError(f"{who}: {fmt!r} is not an MX element format")
    return f


def _here(t: torch.Tensor, dev) -> torch.Tensor:
    """t on dev, contiguous."""
    if t.device != dev:
        t = t.detach().to(dev)
    return t if t.is_contiguous() else t.detach().contiguous()


def _pair(v, f: Format, who: str, what: str):
    """The checked codes and scales of an operand, the codes' shape and K."""
    if not isinstance(v, (tuple, list)) or len(v) != 2 or not isinstance(v[0], torch.Tensor) or \
            not isinstance(v[1], torch.Tensor):
        raise ValueError(f"{who}: {what} must be a pair (codes, scales) of uint8 tensors")
    codes, scales = v
    shape, have = codes.shape, scales.shape
    if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8 or not shape:
        raise ValueError(f"{who}: {what} must be uint8 codes and scales, got {codes.dtype} and {scales.dtype}")
    K = shape[-1] * 2 if f.e + f.m == 3 else shape[-1]
    if K == 0:
        raise ValueError(f"{who}: {what} has no values along its last dimension")
    if len(have) != len(shape) or have[-1] != (K + BLOCK - 1) // BLOCK or have[:-1] != shape[:-1]:
        raise ValueError(f"{who}: scales of {what} must have shape {(*shape[:-1], -(-K // BLOCK))} for {f.name} codes "
                         f"{tuple(shape)}, got {tuple(have)}")
    return codes, scales, shape, K


def _direct(at: int, f: Format, K: int, gathered: bool = False) -> bool:
    """Whether the kernels read contiguous codes at address `at` as they are (else the call lays them out first)."""
    if f.e + f.m == 7:
        return K % 16 == 0 and at % 16 == 0
    return f.e + f.m == 3 and not gathered and K % 128 == 0 and at % 32 == 0


def _room(rows: int, K: int) -> int:
    """The bytes that laying out an operand takes at most: codes and scales at pitches of 16 bytes."""
    return rows * ((K + 15 & -16) + (-(-K // BLOCK) + 15 & -16)) + 128


def lay_packed(w: Pair, fmt: Union[str, Format]) -> Tuple[Pair, str]:
    """(w, fmt) such that the products read w as it is, once for weights that are kept: FP6 codes, and FP4 codes with K
    no multiple of 128, become the E4M3 codes of the same values. Rows that would not be multiples of 16 bytes cannot be
    kept so (the pair has no room between its rows) and come back unchanged."""
    f = _format(fmt, "lay_packed")
    codes, scales, shape, K = _pair(w, f, "lay_packed", "w")
    if f.e + f.m == 7 or K % 16 or (f.e + f.m == 3 and K % 128 == 0):
        return (codes, scales), f.name
    dev = _lib.device_for(codes)
    c = _here(codes, dev)
    wide = torch.empty(*shape[:-1], K, dtype=torch.uint8, device=dev)
    rows = c.numel() // shape[-1]
    if rows:
        _lib.run("mxq_lay_codes", dev, c.data_ptr(), shape[-1], wide.data_ptr(), K, rows, K, f.e, f.m)
    return (_lib.back(wide, codes.device), scales), "MXFP8_E4M3"


def _x_operand(x, x_fmt, who: str, w: torch.Tensor, gathered: bool = False):
    """(data, scales or None, pitch, type, format, bytes of workspace, leading shape, K, device, home) of x: a pair, or a
    float tensor that the call packs."""
    f = _format(x_fmt, who)
    if isinstance(x, torch.Tensor):
        kind = FLOATS.get(x.dtype)
        shape = x.shape
        if kind is None or not shape:
            raise ValueError(f"{who}: x must be a float32, bfloat16 or float16 tensor or a pair (codes, scales), got "
                             f"{x.dtype}")
        K = shape[-1]
        if K == 0:
            raise ValueError(f"{who}: x has no values along its last dimension")
        dev = x.device if x.is_cuda else _lib.device_for(x, w)
        v = x if x.device == dev else x.detach().to(dev)
        if len(shape) != 2:
            v = v.detach().reshape(-1, K)
        rows, stride = v.shape[0], v.stride(0)
        if v.stride(1) != 1 or (rows > 1 and stride < K):
            v = v.detach().contiguous()
            stride = K
        room = _room(rows, K)
        return v, None, stride, 1 + kind, f, room, shape[:-1], K, dev, x.device
    codes, scales, shape, K = _pair(x, f, who, "x")
    dev = codes.device if codes.is_cuda else _lib.device_for(codes, w)
    c, s = _here(codes, dev), _here(scales, dev)
    room = 0 if _direct(c.data_ptr(), f, K, gathered) else _room(c.numel() // shape[-1], K)
    return c, s, shape[-1], 0, f, room, shape[:-1], K, dev, codes.device


def _make_spec(x_e, x_m, w_e, w_m, act, out, out_e, out_m, x_type):
    return _lib.MxqProductSpec(x_e, x_m, w_e, w_m, act, out, out_e, out_m, x_type)


_spec = _lib.cached(_make_spec)


def _w_operand(wc, ws, shape, f: Format, K: int, dev):
    """(codes, scales, bytes of workspace) of w on dev."""
    c, s = _here(wc, dev), _here(ws, dev)
    return c, s, 0 if _direct(c.data_ptr(), f, K) else _room(c.numel() // shape[-1], K)


def _plan_output(out, activation, N: int, who: str):
    """(activation code, output code, output Format or None, F)."""
    if activation is not None and not (isinstance(activation, str) and activation in ACTIVATIONS):
        raise ValueError(f"{who}: activation must be one of {ACTIVATIONS}, got {activation!r}")
    act, F = ACTIVATIONS.index(activation), N
    if act >= FIRST_GATED:
        if N % 2:
            raise ValueError(f"{who}: {activation} needs an even number of rows of w, got {N}")
        F = N // 2
    if isinstance(out, torch.dtype):
        kind = FLOATS.get(out)
        if kind is None:
            raise ValueError(f"{who}: out must be float32, bfloat16, float16 or an MX format, got {out}")
        return act, kind, None, F
    f = _format(out, who)
    if f.e + f.m == 3 and F % 2:
        raise ValueError(f"{who}: packed FP4 pairs up along the output, whose width is {F}")
    return act, PACKED, f, F


def _outputs(lead, out, f, F: int, dev):
    """The empty output: (tensor for the codes or values, scales or None)."""
    if f is None:
        return torch.empty(*lead, F, dtype=out, device=dev), None
    return (torch.empty(*lead, F // 2 if f.e + f.m == 3 else F, dtype=torch.uint8, device=dev),
            torch.empty(*lead, -(-F // BLOCK), dtype=torch.uint8, device=dev))


def _given(y, scales, dev, home):
    if home != dev:
        y, scales = y.to(home), None if scales is None else scales.to(home)
    return y if scales is None else (y, scales)


def _ready():
    if _lib._wait_word is None:                             # the kernel's wait-status word, checked by every call
        _lib.wait_word()


class _Product(torch.autograd.Function):
    """A product whose float arguments are part of a graph."""
    @staticmethod
    def forward(ctx, who, call, x, bias, residual):
        ctx.who, ctx.home = who, None if residual is None else residual.device
        return call()

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        for i, what in ((2, "x"), (3, "bias")):
            if ctx.needs_input_grad[i]:
                raise RuntimeError(f"{ctx.who} is inference only: it has no gradient for {what}; detach it, or call under "
                                   "torch.no_grad()")
        return None, None, None, None, dy.to(ctx.home)


def linear_packed(x: Union[Pair, torch.Tensor], w: Pair, fmt: Union[str, Format], x_fmt: Union[str, Format] = "MXFP8_E4M3",
                  bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                  residual: Optional[torch.Tensor] = None, out: Union[torch.dtype, str] = torch.bfloat16):
    """y = act(x wᵀ + bias) [* up] + residual. x: (... x K) packed to x_fmt (a pair) or floats; w: an N x K pair of
    `fmt`; bias: N values; residual: y's shape and dtype. Returns y (... x F) of dtype `out`, or its (codes, scales)."""
    if isinstance(out, torch.dtype) and _lib.tracked(x, bias, residual):
        return _Product.apply("linear_packed", lambda: _linear(x, w, fmt, x_fmt, bias, activation, residual, out),
                              x if isinstance(x, torch.Tensor) else None, bias, residual)
    return _linear(x, w, fmt, x_fmt, bias, activation, residual, out)


def _linear(x, w, fmt, x_fmt, bias, activation, residual, out):
    who = "linear_packed"
    fw = _format(fmt, who)
    wc, ws, wshape, K = _pair(w, fw, who, "w")
    if len(wshape) != 2:
        raise ValueError(f"{who}: w must be 2-D (N x K), got codes {tuple(wshape)}")
    N = wshape[0]
    act, otype, fo, F = _plan_output(out, activation, N, who)
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"{who}: bias must have shape {(N,)}, got {tuple(bias.shape)}")
    _ready()
    xc, xs, xp, xt, fx, room, lead, Kx, dev, home = _x_operand(x, x_fmt, who, wc)
    if Kx != K:
        raise ValueError(f"{who}: x has {Kx} values per row and w {K}")
    y, ys = _outputs(lead, out, fo, F, dev)
    M = lead[0] if len(lead) == 1 else lead.numel()
    r, r_at, r_stride = None, 0, 0
    if residual is not None:
        if fo is not None:
            raise ValueError(f"{who}: a packed output takes no residual")
        if residual.shape != y.shape or residual.dtype is not out:
            raise ValueError(f"{who}: residual must be {out} of shape {tuple(y.shape)}, got {residual.dtype} "
                             f"{tuple(residual.shape)}")
        r = residual if residual.device == dev else residual.detach().to(dev)
        if len(lead) != 1:
            r = r.detach().reshape(M, F)
        r_stride = r.stride(0)
        if F > 1 and r.stride(1) != 1:
            r = r.detach().contiguous()
            r_stride = F
        r_at = r.data_ptr()
    if M == 0 or N == 0:
        return _given(y, ys, dev, home)
    b = None if bias is None else _lib.on(bias, dev)
    wc, ws, more = _w_operand(wc, ws, wshape, fw, K, dev)
    room += more
    space = torch.empty(room, dtype=torch.uint8, device=dev) if room else None
    spec = _spec(fx.e, fx.m, fw.e, fw.m, act, otype, fo.e if fo else 0, fo.m if fo else 0, xt)
    _lib.run("mxq_linear_packed", dev, xc.data_ptr(), None if xs is None else xs.data_ptr(), xp, M, wc.data_ptr(), ws.data_ptr(), wshape[-1], N, K,
             ctypes.byref(spec), None if b is None else b.data_ptr(), r_at, r_stride, y.data_ptr(),
             None if ys is None else ys.data_ptr(), None if space is None else space.data_ptr(), room)
    return _given(y, ys, dev, home)


def _index(t: torch.Tensor, dev, who: str, what: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32:
        raise ValueError(f"{who}: {what} must be an int32 tensor, got {getattr(t, 'dtype', type(t))}")
    return _here(t, dev)


def experts_packed(x: Union[Pair, torch.Tensor], w: Pair, fmt: Union[str, Format], plan: Dispatch, gather: bool = True,
                   x_fmt: Union[str, Format] = "MXFP8_E4M3", bias: Optional[torch.Tensor] = None,
                   activation: Optional[str] = None, out: Union[torch.dtype, str] = torch.bfloat16):
    """linear_packed by expert: row r of the result belongs to the slot plan.order[r] and is multiplied with its expert's
    weights. w: an E x N x K pair; bias: E x N. x: T x K, a row per token, read through the plan (gather), or
    slots x K in the plan's order (not gather). Returns slots x F in the plan's order; the rows of places without a slot
    (from offsets[-1] on) are not written."""
    if isinstance(out, torch.dtype) and _lib.tracked(x, bias):
        return _Product.apply("experts_packed", lambda: _experts(x, w, fmt, plan, gather, x_fmt, bias, activation, out),
                              x if isinstance(x, torch.Tensor) else None, bias, None)
    return _experts(x, w, fmt, plan, gather, x_fmt, bias, activation, out)


def _experts(x, w, fmt, plan, gather, x_fmt, bias, activation, out):
    who = "experts_packed"
    fw = _format(fmt, who)
    wc, ws, wshape, K = _pair(w, fw, who, "w")
    if len(wshape) != 3:
        raise ValueError(f"{who}: w must be 3-D (experts x N x K), got codes {tuple(wshape)}")
    E, N = wshape[0], wshape[1]
    act, otype, fo, F = _plan_output(out, activation, N, who)
    offsets, order, _ = plan
    if offsets.numel() != E + 1:
        raise ValueError(f"{who}: the plan has {offsets.numel() - 1} experts and w {E}")
    if bias is not None and tuple(bias.shape) != (E, N):
        raise ValueError(f"{who}: bias must have shape {(E, N)}, got {tuple(bias.shape)}")
    _ready()
    xc, xs, xp, xt, fx, room, lead, Kx, dev, home = _x_operand(x, x_fmt, who, wc, gather)
    if Kx != K:
        raise ValueError(f"{who}: x has {Kx} values per row and w {K}")
    if len(lead) != 1:
        raise ValueError(f"{who}: x must be 2-D, got leading shape {tuple(lead)}")
    slots, rows = order.numel(), lead[0]
    if gather:
        if (slots == 0) != (rows == 0) or (rows and slots % rows):
            raise ValueError(f"{who}: {slots} slots are no multiple of x's {rows} rows")
        per = slots // rows if rows else 1
    else:
        if rows != slots:
            raise ValueError(f"{who}: x has {rows} rows and the plan {slots} slots")
        per = 0
    y, ys = _outputs((slots,), out, fo, F, dev)
    if slots == 0 or N == 0 or E == 0:
        return _given(y, ys, dev, home)
    offsets, order = _index(offsets, dev, who, "offsets"), _index(order, dev, who, "order")
    b = None if bias is None else _lib.on(bias, dev)
    wc, ws, more = _w_operand(wc, ws, wshape, fw, K, dev)
    room += more
    if gather and slots > 8 * E:                            # room for x's rows in the plan's order
        room += slots * (-(-K // 16) * 16 + -(-K // BLOCK)) + 256
    space = torch.empty(room, dtype=torch.uint8, device=dev) if room else None
    spec = _spec(fx.e, fx.m, fw.e, fw.m, act, otype, fo.e if fo else 0, fo.m if fo else 0, xt)
    _lib.run("mxq_experts_packed", dev, xc.data_ptr(), None if xs is None else xs.data_ptr(), xp, rows, wc.data_ptr(), ws.data_ptr(), wshape[-1], E, N, K,
             offsets.data_ptr(), order.data_ptr(), slots, per, ctypes.byref(spec), None if b is None else b.data_ptr(),
             y.data_ptr(), None if ys is None else ys.data_ptr(), None if space is None else space.data_ptr(), room)
    return _given(y, ys, dev, home)
