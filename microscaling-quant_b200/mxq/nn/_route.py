"""Routing tokens to experts and adding up what the experts return (no reference counterpart).

    weights, experts = route(logits, k, score="sigmoid", bias=b, groups=8, keep=4, group_score="top2", renormalize=True)
    plan = dispatch(experts, E)                  the slots in the order of their experts
    y = combine(z, weights, plan, residual=r)    y[t] = sum_j weights[t, j] z[plan.where[t, j]] + r[t]

route scores the T x E logits in float32 by softmax or sigmoid. Without a bias the experts are ranked by their logits,
with one by score + bias (the bias balances the choice only; the weights are the plain scores). groups > 1 cuts the
experts into equal runs, of which the `keep` best take part, by their largest ranking value or ("top2") the sum of
their two largest. The k best experts are returned in descending order, every tie going to the lowest index; their
scores are divided by (their sum + 1e-20) if `renormalize` and multiplied with `scale`.

Experts with a logit of -Inf are never chosen: a place with nothing left to choose gets expert -1 and weight 0, and its
slot takes no part in dispatch, the products and combine (a padded token: a row of -Inf). A row that holds a NaN has
weights NaN.

route is differentiable in the logits and combine in z, weights and residual (first order); experts and the plan are
whole numbers and have no gradient. route_backward and combine_backward are the gradients by themselves.
"""
from typing import Optional, Tuple

import ctypes

import torch

from .. import _lib
from ._packed import FLOATS, Dispatch, _index

__all__ = ["route", "route_backward", "dispatch", "combine", "combine_backward"]

SCORES = ("softmax", "sigmoid")
GROUP_SCORES = ("max", "top2")


def _make_spec(score, groups, keep, top2, renormalize, scale):
    return _lib.MxqRouteSpec(score, groups, keep, top2, renormalize, scale)


_spec = _lib.cached(_make_spec)


def _route_args(who, logits, k, score, groups, keep, group_score):
    if not isinstance(logits, torch.Tensor) or logits.dtype not in FLOATS or logits.ndim != 2:
        raise ValueError(f"{who}: logits must be a 2-D float32, bfloat16 or float16 tensor (tokens x experts)")
    E = logits.shape[1]
    if not isinstance(k, int) or not 1 <= k <= min(E, 32):
        raise ValueError(f"{who}: k must be in [1, min(experts, 32)], got {k!r} for {E} experts")
    if score not in SCORES or group_score not in GROUP_SCORES:
        raise ValueError(f"{who}: score must be one of {SCORES} and group_score one of {GROUP_SCORES}, got {score!r} and "
                         f"{group_score!r}")
    if not 1 <= groups <= 32 or E % groups or not 1 <= keep <= groups:
        raise ValueError(f"{who}: cannot keep {keep} of {groups} equal groups of {E} experts")
    if E > 1024:
        raise ValueError(f"{who}: at most 1024 experts, got {E}")


def _rows(t: torch.Tensor, dev) -> torch.Tensor:
    """t on dev with its rows contiguous (any row stride)."""
    t = t.detach().to(dev)
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 and t.is_contiguous() else t.contiguous()


def _route(logits, k, score, bias, groups, keep, group_score, renormalize, scale):
    T, E = logits.shape
    home, dev = logits.device, _lib.device_for(logits)
    l = _rows(logits, dev)
    b = None if bias is None else _lib.on(bias, dev)
    weights = torch.empty((T, k), dtype=torch.float32, device=dev)
    experts = torch.empty((T, k), dtype=torch.int32, device=dev)
    s = _spec(SCORES.index(score), groups, keep, int(group_score == "top2"), int(bool(renormalize)), float(scale))
    _lib.run("mxq_route", dev, _lib.ptr(l), FLOATS[l.dtype], l.stride(0), _lib.ptr(b), _lib.ptr(weights), _lib.ptr(experts),
             T, E, k, ctypes.byref(s))
    return _lib.back(weights, home), _lib.back(experts, home)


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
    _route_args("route", logits, k, score, groups, keep, group_score)
    if bias is not None and tuple(bias.shape) != (logits.shape[1],):
        raise ValueError(f"route: bias must have shape {(logits.shape[1],)}, got {tuple(bias.shape)}")
    if logits.requires_grad and torch.is_grad_enabled():
        return _Route.apply(logits, k, score, bias, groups, keep, group_score, renormalize, scale)
    return _route(logits, k, score, bias, groups, keep, group_score, renormalize, scale)


def route_backward(grad: torch.Tensor, logits: torch.Tensor, experts: torch.Tensor, score: str = "softmax",
                   renormalize: bool = False, scale: float = 1.0) -> torch.Tensor:
    """d loss / d logits, of their shape and dtype, from grad = d loss / d weights and the experts that route chose."""
    who = "route_backward"
    if experts.ndim != 2:
        raise ValueError(f"{who}: experts must be 2-D (tokens x k), got {tuple(experts.shape)}")
    _route_args(who, logits, experts.shape[1], score, 1, 1, "max")
    T, E = logits.shape
    k = experts.shape[1]
    if experts.shape[0] != T or grad.shape != experts.shape:
        raise ValueError(f"{who}: grad {tuple(grad.shape)} and experts {tuple(experts.shape)} must be {T} x k")
    home, dev = logits.device, _lib.device_for(logits)
    l, g, e = _rows(logits, dev), _lib.on(grad, dev), _index(experts, dev, who, "experts")
    out = torch.empty((T, E), dtype=l.dtype, device=dev)
    s = _spec(SCORES.index(score), 1, 1, 0, int(bool(renormalize)), float(scale))
    _lib.run("mxq_route_backward", dev, _lib.ptr(g), _lib.ptr(l), FLOATS[l.dtype], l.stride(0), _lib.ptr(e), _lib.ptr(out),
             T, E, k, ctypes.byref(s))
    return _lib.back(out, home)


def dispatch(experts: torch.Tensor, n_experts: int) -> Dispatch:
    """The slots of experts (T x k, int32) in the order of their experts, each expert's in their own order. A slot whose
    expert is outside [0, n_experts) is left out."""
    if not isinstance(n_experts, int) or not 1 <= n_experts <= 1024:
        raise ValueError(f"dispatch: n_experts must be in [1, 1024], got {n_experts!r}")
    home, dev = experts.device, _lib.device_for(experts)
    e = _index(experts, dev, "dispatch", "experts")
    offsets = torch.empty(n_experts + 1, dtype=torch.int32, device=dev)
    order = torch.empty(e.numel(), dtype=torch.int32, device=dev)
    where = torch.empty(e.shape, dtype=torch.int32, device=dev)
    _lib.run("mxq_dispatch", dev, _lib.ptr(e), e.numel(), n_experts, _lib.ptr(offsets), _lib.ptr(order), _lib.ptr(where))
    return Dispatch(_lib.back(offsets, home), _lib.back(order, home), _lib.back(where, home))


def _combine_args(who, z, weights, plan):
    if not isinstance(z, torch.Tensor) or z.dtype not in FLOATS or z.ndim != 2:
        raise ValueError(f"{who}: z must be a 2-D float32, bfloat16 or float16 tensor (slots x N)")
    if weights.ndim != 2 or weights.shape != plan.where.shape or plan.order.numel() != plan.where.numel():
        raise ValueError(f"{who}: weights {tuple(weights.shape)} do not match the plan's {tuple(plan.where.shape)} slots")
    if z.shape[0] != plan.where.numel():
        raise ValueError(f"{who}: z has {z.shape[0]} rows and the plan {plan.where.numel()} slots")


def _combine(z, weights, where, residual):
    (T, k), N = where.shape, z.shape[1]
    home, dev = z.device, _lib.device_for(z)
    zc = z.detach().to(dev).contiguous()
    w, at = _lib.on(weights, dev), _index(where, dev, "combine", "where")
    r = None if residual is None else _rows(residual, dev)
    y = torch.empty((T, N), dtype=z.dtype, device=dev)
    if k == 0:
        return y.zero_() if residual is None else y.copy_(residual)
    _lib.run("mxq_combine", dev, _lib.ptr(zc), FLOATS[zc.dtype], _lib.ptr(w), _lib.ptr(at), _lib.ptr(r),
             r.stride(0) if r is not None else 0, _lib.ptr(y), T, k, N)
    return _lib.back(y, home)


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
    _combine_args("combine", z, weights, plan)
    T, N = plan.where.shape[0], z.shape[1]
    if residual is not None and (tuple(residual.shape) != (T, N) or residual.dtype != z.dtype):
        raise ValueError(f"combine: residual must be {z.dtype} of shape {(T, N)}, got {residual.dtype} "
                         f"{tuple(residual.shape)}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (z, weights, residual)):
        return _Combine.apply(z, weights, *plan, residual)
    return _combine(z, weights, plan.where, residual)


def combine_backward(dy: torch.Tensor, z: torch.Tensor, weights: torch.Tensor,
                     plan: Dispatch) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dz, dw) of combine: dz[place] = weights[slot] dy[t] (0 at the places without a slot), dw[t, j] = dy[t] . z[place]
    in float32 (0 for a slot left out)."""
    who = "combine_backward"
    _combine_args(who, z, weights, plan)
    (T, k), N = plan.where.shape, z.shape[1]
    if tuple(dy.shape) != (T, N) or dy.dtype != z.dtype:
        raise ValueError(f"{who}: dy must be {z.dtype} of shape {(T, N)}, got {dy.dtype} {tuple(dy.shape)}")
    home, dev = z.device, _lib.device_for(z)
    zc, g = z.detach().to(dev).contiguous(), _rows(dy, dev)
    w, at, order = _lib.on(weights, dev), _index(plan.where, dev, who, "where"), _index(plan.order, dev, who, "order")
    dz = torch.empty((T * k, N), dtype=z.dtype, device=dev)
    dw = torch.empty((T, k), dtype=torch.float32, device=dev)
    if T and k:
        _lib.run("mxq_combine_backward", dev, _lib.ptr(g), g.stride(0), _lib.ptr(zc), FLOATS[zc.dtype], _lib.ptr(w),
                 _lib.ptr(at), _lib.ptr(order), _lib.ptr(dz), _lib.ptr(dw), T, k, N)
    return _lib.back(dz, home), _lib.back(dw, home)
