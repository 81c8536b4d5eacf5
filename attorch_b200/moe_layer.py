"""
``MixtureOfExperts``: the transformer block's MLP (examples/wikitext-2/gpt.py:30-37 of the reference) with a
weight per expert: gate, routing, dispatch, up-projection with its fused activation, down-projection, combine.  A
forward pass of up to 256 tokens is six launches (seven when gated), none of which the host waits for.
"""

from typing import Optional

import torch
from torch import Tensor, nn

from .expert_routing_layer import Router, combine, dispatch
from .float8_linear_layer import Float8GroupedLinear
from .glu_layer import GLU
from .grouped_linear_layer import GroupedLinear


class MixtureOfExperts(nn.Module):
    """
    Sends every token through ``top_k`` of ``num_experts`` MLPs and sums their outputs by the router's weights.

    Args:
        dim: Number of input and output features.
        hidden: Number of features between an expert's two projections.
        num_experts: Number of experts, at most 512.
        top_k: Experts a token, at most 32.
        act_func: Activation of the up-projection, as ``Linear``.
        gated: Flag for a gated up-projection: ``x1 * act(x2)`` of a projection twice as wide, as ``GLU``.
        bias: Flag for additive biases in the experts.
        score_func: 'softmax' or 'sigmoid', as ``route``.
        renormalize: Flag for dividing a token's weights by their sum.
        device: Device to use.
        dtype: Dtype of layer.
    """
    def __init__(self, dim: int, hidden: int, num_experts: int, top_k: int, act_func: str = 'gelu', gated: bool = False,
                 bias: bool = True, score_func: str = 'softmax', renormalize: bool = True, device='cuda',
                 dtype: torch.dtype = torch.float32) -> None:
        super().__init__()
        self.router = Router(dim, num_experts, top_k, score_func, renormalize, device, dtype)
        self.up = GroupedLinear(num_experts, dim, 2 * hidden if gated else hidden, bias, None if gated else act_func, device, dtype)
        self.glu = GLU(-1, act_func) if gated else None
        self.down = GroupedLinear(num_experts, hidden, dim, bias, None, device, dtype)

    def to_float8(self) -> 'MixtureOfExperts':
        """Replaces the experts' weights by their 8-bit form, for serving (no gradient); returns the layer."""
        if isinstance(self.up, GroupedLinear):
            self.up = Float8GroupedLinear.from_grouped(self.up)
            self.down = Float8GroupedLinear.from_grouped(self.down)
        return self

    def forward(self, input: Tensor, mask: Optional[Tensor] = None) -> Tensor:
        """``input``: ``[..., dim]``; ``mask``: optional ``[...]`` boolean, False for padding, whose output is
        zero and whose values, NaN among them, reach no gradient of the parameters."""
        tokens = input.flatten(0, -2)
        routing = self.router(tokens, None if mask is None else mask.flatten())
        rows = self.up(dispatch(tokens, routing), routing.offsets)
        if self.glu is not None:
            rows = self.glu(rows)
        rows = self.down(rows, routing.offsets)
        return combine(rows, routing).view(input.shape)
