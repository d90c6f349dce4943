"""Routing tokens to experts and adding up what the experts return (no reference counterpart).

    weights, experts = route(logits, k, score="sigmoid", bias=b, groups=8, keep=4, group_score="top2", renormalize=True)
    plan = dispatch(experts, E)                  the slots in the order of their experts
    y = combine(z, weights, plan, residual=r)    y[t] = sum_j weights[t, j] z[plan.where[t, j]] + r[t]

route scores the T x E logits in float32 by softmax or sigmoid. Without a bias the experts are ranked by their logits,
with one by score + bias (the bias balances the choice only; the weights are the plain scores). groups > 1 cuts the
experts into equal runs, of which the `keep` best take part, by their largest ranking value or ("top2") the sum of
their two largest scores, or score + bias (an expert with a logit of -Inf counts there with the score 0 that it has; a run with
nobody to choose takes no part). The k best experts are returned in descending order, every tie going to the lowest index; their
scores are divided by (their sum + 1e-20) if `renormalize` and multiplied with `scale`.

Experts with a logit of -Inf are never chosen: a place with nothing left to choose gets expert -1 and weight 0, and its
slot takes no part in dispatch, the products and combine (a padded token: a row of -Inf). A row that holds a NaN, or
under softmax a +Inf, has weights NaN, and so has its gradient.

route is differentiable in the logits and combine in z, weights and residual (first order); experts and the plan are
whole numbers and have no gradient; forward-mode tangents raise. route_backward and combine_backward are the gradients by themselves.
"""
from typing import Optional, Tuple

import ctypes

import torch

from .. import _lib
from ._packed import FLOATS, Dispatch, _here, _index

__all__ = ["route", "route_backward", "dispatch", "combine", "combine_backward"]

SCORES = ("softmax", "sigmoid")
GROUP_SCORES = ("max", "top2")
#: slots up to which dispatch needs no workspace
ONE_LAUNCH = 98304


def _make_spec(score, groups, keep, top2, renormalize, scale):
    return _lib.MxqRouteSpec(score, groups, keep, top2, renormalize, scale)


_spec = _lib.cached(_make_spec)


def _route_args(who, logits, k, score, groups, keep, group_score):
    """(tokens, experts) of checked arguments."""
    if not isinstance(logits, torch.Tensor) or logits.dtype not in FLOATS or logits.dim() != 2:
        raise ValueError(f"{who}: logits must be a 2-D float32, bfloat16 or float16 tensor (tokens x experts)")
    T, E = logits.shape
    if not isinstance(k, int) or not 1 <= k <= min(E, 32):
        raise ValueError(f"{who}: k must be in [1, min(experts, 32)], got {k!r} for {E} experts")
    if score not in SCORES or group_score not in GROUP_SCORES:
        raise ValueError(f"{who}: score must be one of {SCORES} and group_score one of {GROUP_SCORES}, got {score!r} and "
                         f"{group_score!r}")
    if not 1 <= groups <= 32 or E % groups or not 1 <= keep <= groups:
        raise ValueError(f"{who}: cannot keep {keep} of {groups} equal groups of {E} experts")
    if E > 1024:
        raise ValueError(f"{who}: at most 1024 experts, got {E}")
    return T, E


def _rows(t: torch.Tensor, dev) -> torch.Tensor:
    """t (2-D) on dev with its rows contiguous (any row stride)."""
    if t.device != dev:
        t = t.detach().to(dev)
    return t if t.is_contiguous() or t.stride(1) == 1 else t.detach().contiguous()


def _device(t: torch.Tensor):
    return t.device if t.is_cuda else _lib.device_for(t)


def _route(logits, k, score, bias, groups, keep, group_score, renormalize, scale):
    T, E = logits.shape
    home, dev = logits.device, _device(logits)
    l = _rows(logits, dev)
    b = None if bias is None else _lib.on(bias, dev)
    weights = torch.empty(T, k, dtype=torch.float32, device=dev)
    experts = torch.empty(T, k, dtype=torch.int32, device=dev)
    s = _spec(SCORES.index(score), groups, keep, int(group_score == "top2"), int(bool(renormalize)), float(scale))
    _lib.run("mxq_route", dev, l.data_ptr(), FLOATS[l.dtype], l.stride(0), None if b is None else b.data_ptr(),
             weights.data_ptr(), experts.data_ptr(), T, E, k, ctypes.byref(s))
    if home == dev:
        return weights, experts
    return weights.to(home), experts.to(home)


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, score, bias, groups, keep, group_score, renormalize, scale):
        weights, experts = _route(logits, k, score, bias, groups, keep, group_score, renormalize, scale)
        ctx.save_for_backward(logits, experts)
        ctx.how = score, renormalize, scale
        ctx.mark_non_differentiable(experts)
        return weights, experts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        logits, experts = ctx.saved_tensors
        score, renormalize, scale = ctx.how
        return (route_backward(grad, logits, experts, score, renormalize, scale), *(None,) * 8)


def route(logits: torch.Tensor, k: int, score: str = "softmax", bias: Optional[torch.Tensor] = None, groups: int = 1,
          keep: int = 1, group_score: str = "max", renormalize: bool = False,
          scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """The k experts of each token: (weights T x k float32, experts T x k int32), as the module's text says."""
    _, E = _route_args("route", logits, k, score, groups, keep, group_score)
    if bias is not None and tuple(bias.shape) != (E,):
        raise ValueError(f"route: bias must have shape {(E,)}, got {tuple(bias.shape)}")
    if _lib.tracked(logits):
        return _Route.apply(logits, k, score, bias, groups, keep, group_score, renormalize, scale)
    return _route(logits, k, score, bias, groups, keep, group_score, renormalize, scale)


def route_backward(grad: torch.Tensor, logits: torch.Tensor, experts: torch.Tensor, score: str = "softmax",
                   renormalize: bool = False, scale: float = 1.0) -> torch.Tensor:
    """d loss / d logits, of their shape and dtype, from grad = d loss / d weights and the experts that route chose."""
    who = "route_backward"
    if experts.ndim != 2:
        raise ValueError(f"{who}: experts must be 2-D (tokens x k), got {tuple(experts.shape)}")
    k = experts.shape[1]
    T, E = _route_args(who, logits, k, score, 1, 1, "max")
    if experts.shape[0] != T or grad.shape != experts.shape:
        raise ValueError(f"{who}: grad {tuple(grad.shape)} and experts {tuple(experts.shape)} must be {T} x k")
    home, dev = logits.device, _device(logits)
    l, g, e = _rows(logits, dev), _lib.on(grad, dev), _index(experts, dev, who, "experts")
    out = torch.empty(T, E, dtype=l.dtype, device=dev)
    s = _spec(SCORES.index(score), 1, 1, 0, int(bool(renormalize)), float(scale))
    _lib.run("mxq_route_backward", dev, g.data_ptr(), l.data_ptr(), FLOATS[l.dtype], l.stride(0), e.data_ptr(),
             out.data_ptr(), T, E, k, ctypes.byref(s))
    return _lib.back(out, home)


def dispatch(experts: torch.Tensor, n_experts: int) -> Dispatch:
    """The slots of experts (T x k, int32) in the order of their experts, each expert's in their own order. A slot whose
    expert is outside [0, n_experts) is left out."""
    if not isinstance(n_experts, int) or not 1 <= n_experts <= 1024:
        raise ValueError(f"dispatch: n_experts must be in [1, 1024], got {n_experts!r}")
    home, dev = experts.device, _device(experts)
    e = _index(experts, dev, "dispatch", "experts")
    n = e.numel()
    offsets = torch.empty(n_experts + 1, dtype=torch.int32, device=dev)
    order = torch.empty(n, dtype=torch.int32, device=dev)
    where = torch.empty_like(e)
    room, space = 0, None
    if n > ONE_LAUNCH:
        with _lib.using(dev):                               # the size goes by the device's SMs
            room = _lib.lib().mxq_dispatch_workspace(n, n_experts)
        space = torch.empty(room, dtype=torch.uint8, device=dev)
    _lib.run("mxq_dispatch", dev, e.data_ptr(), n, n_experts, offsets.data_ptr(), order.data_ptr(), where.data_ptr(),
             None if space is None else space.data_ptr(), room)
    if home != dev:
        offsets, order, where = offsets.to(home), order.to(home), where.to(home)
    return Dispatch(offsets, order, where)


def _combine_args(who, z, weights, plan):
    """(T, k, N) of checked arguments."""
    if not isinstance(z, torch.Tensor) or z.dtype not in FLOATS or z.dim() != 2:
        raise ValueError(f"{who}: z must be a 2-D float32, bfloat16 or float16 tensor (slots x N)")
    _, order, where = plan
    shape = where.shape
    if len(shape) != 2 or weights.shape != shape or order.numel() != shape[0] * shape[1]:
        raise ValueError(f"{who}: weights {tuple(weights.shape)} do not match the plan's {tuple(shape)} slots")
    slots, N = z.shape
    if slots != shape[0] * shape[1]:
        raise ValueError(f"{who}: z has {slots} rows and the plan {shape[0] * shape[1]} slots")
    return shape[0], shape[1], N


def _combine(z, weights, where, residual):
    (T, k), N = where.shape, z.shape[1]
    home, dev = z.device, _device(z)
    zc, w, at = _here(z, dev), _lib.on(weights, dev), _index(where, dev, "combine", "where")
    r = None if residual is None else _rows(residual, dev)
    y = torch.empty(T, N, dtype=z.dtype, device=dev)
    if k == 0:
        y = y.zero_() if r is None else y.copy_(r.detach())
    else:
        _lib.run("mxq_combine", dev, zc.data_ptr(), FLOATS[zc.dtype], w.data_ptr(), at.data_ptr(),
                 None if r is None else r.data_ptr(), 0 if r is None else r.stride(0), y.data_ptr(), T, k, N)
    return y if home == dev else y.to(home)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, weights, offsets, order, where, residual):
        ctx.save_for_backward(z, weights, offsets, order, where)
        ctx.residual = residual is not None
        return _combine(z, weights, where, residual)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        z, weights, *plan = ctx.saved_tensors
        dz, dw = combine_backward(dy, z, weights, Dispatch(*plan))
        return dz, dw.to(weights.dtype), None, None, None, dy if ctx.residual else None


def combine(z: torch.Tensor, weights: torch.Tensor, plan: Dispatch, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] = sum_j weights[t, j] z[plan.where[t, j]] (+ residual[t]), of z's dtype, summed in float32 in the order of j.
    z: slots x N in the plan's order. A slot left out adds its weight times 0."""
    T, _, N = _combine_args("combine", z, weights, plan)
    if residual is not None and (tuple(residual.shape) != (T, N) or residual.dtype != z.dtype):
        raise ValueError(f"combine: residual must be {z.dtype} of shape {(T, N)}, got {residual.dtype} "
                         f"{tuple(residual.shape)}")
    if _lib.tracked(z, weights, residual):
        return _Combine.apply(z, weights, *plan, residual)
    return _combine(z, weights, plan.where, residual)


def combine_backward(dy: torch.Tensor, z: torch.Tensor, weights: torch.Tensor,
                     plan: Dispatch) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dz, dw) of combine: dz[place] = weights[slot] dy[t] (0 at the places without a slot), dw[t, j] = dy[t] . z[place]
    in float32 (0 for a slot left out)."""
    who = "combine_backward"
    T, k, N = _combine_args(who, z, weights, plan)
    if tuple(dy.shape) != (T, N) or dy.dtype != z.dtype:
        raise ValueError(f"{who}: dy must be {z.dtype} of shape {(T, N)}, got {dy.dtype} {tuple(dy.shape)}")
    home, dev = z.device, _device(z)
    zc, g = _here(z, dev), _rows(dy, dev)
    w, at, order = _lib.on(weights, dev), _index(plan.where, dev, who, "where"), _index(plan.order, dev, who, "order")
    dz = torch.empty(T * k, N, dtype=z.dtype, device=dev)
    dw = torch.empty(T, k, dtype=torch.float32, device=dev)
    if T and k:
        _lib.run("mxq_combine_backward", dev, g.data_ptr(), g.stride(0), zc.data_ptr(), FLOATS[zc.dtype], w.data_ptr(),
                 at.data_ptr(), order.data_ptr(), dz.data_ptr(), dw.data_ptr(), T, k, N)
    if home == dev:
        return dz, dw
    return dz.to(home), dw.to(home)
