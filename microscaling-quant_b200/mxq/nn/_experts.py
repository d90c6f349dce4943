"""MXExperts: the experts of a mixture-of-experts layer on packed MX weights (no reference counterpart).

    layer = MXExperts(gate_up, down, "MXFP8_E4M3")               E x 2F x H, E x H x F
    weights, experts = nn.route(x @ router.T, k, renormalize=True)
    y = layer(x, weights, experts, residual=x)

forward: the plan of the slots, the gated up-projection with x packed and read through the plan and its output packed
again, the down-projection, the weighted sum. The weights are packed once by block.ocp (`fmt`), activations to `act_fmt`
in each call. The packed weights are the layer's state: state_dict has their codes and scales, and their formats, which a layer
that loads them takes over. Differentiable in `weights` and `residual` (a router tuned against the packed experts); x and the experts
themselves have no gradient.
"""
from typing import Optional, Union

import torch
from torch import nn

from ..block import ocp
from ..element_quant.formats import FORMATS, Format, get
from ._packed import GATED, experts_packed, lay_packed
from ._route import combine, dispatch

__all__ = ["MXExperts"]


class MXExperts(nn.Module):
    def __init__(self, gate_up: torch.Tensor, down: torch.Tensor, fmt: Union[str, Format] = "MXFP8_E4M3",
                 act_fmt: Union[str, Format] = "MXFP8_E4M3", activation: str = "swiglu"):
        super().__init__()
        if gate_up.ndim != 3 or down.ndim != 3 or gate_up.shape[0] != down.shape[0] or \
                gate_up.shape[1] != 2 * down.shape[2] or gate_up.shape[2] != down.shape[1]:
            raise ValueError(f"MXExperts: gate_up must be E x 2F x H and down E x H x F, got {tuple(gate_up.shape)} and "
                             f"{tuple(down.shape)}")
        if activation not in GATED:
            raise ValueError(f"MXExperts: activation must be one of {GATED}, got {activation!r}")
        if get(fmt) is None or get(act_fmt) is None:
            raise ValueError("MXExperts: fmt and act_fmt must be MX element formats")
        self.n_experts, self.hidden, self.inner = gate_up.shape[0], gate_up.shape[2], down.shape[2]
        self.act_fmt, self.activation = get(act_fmt).name, activation
        for name, w in (("up", gate_up), ("down", down)):
            (codes, scales), self_fmt = lay_packed(ocp.quantize_packed(w.detach().float(), fmt, axis=-1), fmt)
            self.register_buffer(f"{name}_codes", codes)
            self.register_buffer(f"{name}_scales", scales)
            setattr(self, f"{name}_fmt", self_fmt)

    def get_extra_state(self) -> torch.Tensor:
        """(exponent, mantissa) bits of the up and the down weights' codes: a tensor, as all of a state_dict."""
        return torch.tensor([(FORMATS[f].e, FORMATS[f].m) for f in (self.up_fmt, self.down_fmt)], dtype=torch.uint8)

    def set_extra_state(self, state: torch.Tensor):
        names = {(f.e, f.m): f.name for f in FORMATS.values()}
        self.up_fmt, self.down_fmt = (names[tuple(em)] for em in state.tolist())

    def forward(self, x: torch.Tensor, weights: torch.Tensor, experts: torch.Tensor,
                residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x (... x H) with each token's weights and experts (tokens x k, as nn.route gives them)."""
        flat = x.detach().reshape(-1, self.hidden)
        if tuple(experts.shape) != tuple(weights.shape) or experts.ndim != 2 or experts.shape[0] != flat.shape[0]:
            raise ValueError(f"MXExperts: weights {tuple(weights.shape)} and experts {tuple(experts.shape)} must be "
                             f"{flat.shape[0]} x k")
        plan = dispatch(experts, self.n_experts)
        h = experts_packed(flat, (self.up_codes, self.up_scales), self.up_fmt, plan, x_fmt=self.act_fmt,
                           activation=self.activation, out=self.act_fmt)
        z = experts_packed(h, (self.down_codes, self.down_scales), self.down_fmt, plan, gather=False, x_fmt=self.act_fmt,
                           out=x.dtype)
        r = None if residual is None else residual.reshape(-1, self.hidden)
        return combine(z, weights, plan, residual=r).reshape(x.shape)

    def extra_repr(self) -> str:
        return (f"experts={self.n_experts}, hidden={self.hidden}, inner={self.inner}, fmt={self.up_fmt!r}, "
                f"act_fmt={self.act_fmt!r}, activation={self.activation!r}")
