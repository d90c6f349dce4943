"""mxq.nn — putting Schemes into a model.

    MXLinear(linear, scheme)     one nn.Linear computed through one Scheme (inference only)
    patch(model, rules)          a Scheme per layer name or type (first matching rule wins); (qk, pv) pairs route an
                                 attention module's core through attend
    is_attention                 a selector for the attention projections
    attend(q, k, v, mask, scale, qk, pv)   the attention core with Q·Kᵀ and P·V through two Schemes

and the feed-forward on packed MX operands, on the tensor cores (no reference counterpart):

    linear_packed(x, w, fmt, ...)         act(x wᵀ + bias) [* up] + residual, the output a float tensor or packed again
    experts_packed(x, w, fmt, plan, ...)  the same by expert, rows in the plan's order
    lay_packed(w, fmt)                    weights laid out once as the products read them
    route(logits, k, ...), dispatch(experts, n)     the experts of each token; the slots in the order of their experts
    combine(z, weights, plan, ...)        the weighted sum of the experts' rows
    route_backward, combine_backward      their gradients (route and combine are differentiable as they are)
    MXExperts(gate_up, down, fmt)         all of it as one layer
"""
from ._attention import attend
from ._experts import MXExperts
from ._linear import MXLinear
from ._packed import Dispatch, experts_packed, lay_packed, linear_packed
from ._patch import is_attention, patch
from ._route import combine, combine_backward, dispatch, route, route_backward

__all__ = ["MXLinear", "patch", "is_attention", "attend", "linear_packed", "experts_packed", "lay_packed", "Dispatch",
           "route", "route_backward", "dispatch", "combine", "combine_backward", "MXExperts"]
