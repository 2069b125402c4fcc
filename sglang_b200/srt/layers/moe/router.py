"""The router in front of the routed experts: logits of the hidden states, then experts and weights from them."""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from .token_dispatcher import StandardTopKOutput
from .topk import route_experts


class Router(nn.Module):
    """`forward(hidden_states)` -> what `FusedMoE` takes.  The product keeps float32 logits (`ops.router_logits`), which decide as they are
    (`ops.route_topk`, whose arguments the others are)."""

    def __init__(self, num_experts: int, hidden_size: int, top_k: int, scoring_func: str = "softmax", renormalize: bool = True,
                 num_expert_group: int = 1, topk_group: int = 1, group_top: Optional[int] = None, use_correction_bias: bool = False,
                 routed_scaling_factor: float = 1.0, params_dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        self.top_k, self.renormalize, self.scoring_func = top_k, renormalize, scoring_func
        self.num_expert_group, self.topk_group, self.group_top = num_expert_group, topk_group, group_top
        self.routed_scaling_factor = routed_scaling_factor
        self.weight = nn.Parameter(torch.empty(num_experts, hidden_size, dtype=params_dtype, device=device), requires_grad=False)
        self.correction_bias = nn.Parameter(torch.zeros(num_experts, dtype=torch.float32, device=device),
                                            requires_grad=False) if use_correction_bias else None

    def forward(self, hidden_states: torch.Tensor) -> StandardTopKOutput:
        from .... import ops

        logits = ops.router_logits(hidden_states, self.weight)
        weights, ids = route_experts(logits, self.top_k, self.renormalize, self.num_expert_group, self.topk_group, self.scoring_func,
                                     self.correction_bias, self.routed_scaling_factor, self.group_top)
        return StandardTopKOutput(weights, ids, logits)
