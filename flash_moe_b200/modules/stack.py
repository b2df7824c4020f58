"""A residual stack of FlashMoE layers used as the MLP path of a decoder: x <- x + layer(x).

The reference ships the single layer only; this is the caller-side composition of the
multi-layer benchmark configuration (layer l seeded with torch.manual_seed(l)).  The skip connection is
handed to the layer (`residual=`), which adds it in the epilogue of its last GEMM: one kernel fewer per
layer and one rounding of `x + layer(x)` instead of two.  With `pre_norm=True` each layer sees
`rms_norm(x)` (a learnable weight per layer) while the skip connection carries the un-normalised x - the
usual pre-norm decoder block.  `GraphedFlashMoE(stack, x)` captures the whole stack in one CUDA graph.

`fused_norm=True` (with `pre_norm`) takes skip connection and norm between two layers of a training step in one kernel each way
(`add_rms_norm`) instead of torch's addition and rms_norm; the sums are rounded alike, the normalised values and gradients agree
to within their rounding.  Under autocast, or with norm weights of another dtype, torch's functions stay.  `balance_loss` and
`clip_grad_norm_` are what a training step needs beside the layers."""

from __future__ import annotations

from typing import List, Optional, Tuple, Union

import torch
import torch.nn as nn

from .. import _lib
from .flash_moe import FlashMoE, FlashMoEConfig


class FlashMoEStack(nn.Module):
    fused_norm = False  # of the class, for stacks that were pickled without it

    def __init__(self, config: FlashMoEConfig, num_layers: int, seeds=None, pre_norm: bool = False, norm_eps: float = 1e-6,
                 fused_norm: bool = False):
        super().__init__()
        self.norm_eps = norm_eps
        self.fused_norm = fused_norm
        self.norms = (nn.ParameterList([nn.Parameter(torch.ones(config.hidden_size)) for _ in range(num_layers)])
                      if pre_norm else None)
        layers = []
        for i in range(num_layers):
            if seeds is not None:
                torch.manual_seed(seeds[i])
            layers.append(FlashMoE(config))
        self.layers = nn.ModuleList(layers)
        # the layers run one after another on one stream, so they can share one scratch allocation
        for layer in layers[1:]:
            layer._workspaces = layers[0]._workspaces

    def forward(self, hidden_states: torch.Tensor, return_routing: bool = False) -> Tuple[torch.Tensor, List[torch.Tensor]]:
        """Returns the final hidden states and every layer's router logits.  ``return_routing=True`` keeps every layer's
        selected ids and gates in its ``last_indices`` / ``last_gates``."""
        # handed on only where it is asked for: a layer that a caller put here may not know it
        routing = {"return_routing": True} if return_routing else {}
        if self.norms is not None and self.fused_norm and torch.is_grad_enabled() and not torch.is_autocast_enabled("cuda") \
                and all(w.dtype == hidden_states.dtype for w in self.norms) \
                and (hidden_states.requires_grad or any(p.requires_grad for p in self.parameters())):
            return self._forward_fused_norm(hidden_states, routing)
        all_logits = []
        x = hidden_states
        for i, layer in enumerate(self.layers):
            if self.norms is not None:
                if torch.is_grad_enabled() and (x.requires_grad or self.norms[i].requires_grad):
                    xn = torch.nn.functional.rms_norm(x, (x.shape[-1],), self.norms[i], self.norm_eps)
                else:
                    from ..ops.rms_norm import rms_norm

                    xn = rms_norm(x, self.norms[i].detach(), self.norm_eps)
                x, logits = layer(xn, residual=x, **routing)
            else:
                x, logits = layer(x, residual=x, **routing)
            all_logits.append(logits)
        return x, all_logits

    def _forward_fused_norm(self, x, routing):
        from ..ops.add_rms_norm import add_rms_norm

        all_logits, y = [], None
        for layer, weight in zip(self.layers, self.norms):
            if y is None:
                xn, x = add_rms_norm(x, None, weight, self.norm_eps)
            else:
                xn, x = add_rms_norm(y, x, weight, self.norm_eps)
            y, logits = layer(xn, **routing)
            all_logits.append(logits)
        return (x if y is None else x + y), all_logits

    def balance_loss(self, all_logits: List[torch.Tensor], token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Mean over the layers of `FlashMoE.balance_loss` for the logits that a forward with ``return_routing=True`` returned."""
        if len(all_logits) != len(self.layers) or not self.layers:
            raise _lib.FmoeError("expected the router logits of every layer")
        losses = [layer.balance_loss(logits, token_mask) for layer, logits in zip(self.layers, all_logits)]
        return torch.stack(losses).mean() if len(losses) > 1 else losses[0]

    def clip_grad_norm_(self, max_norm: float, grad_scale: Union[float, torch.Tensor] = 1.0) -> torch.Tensor:
        """`flash_moe_b200.clip_grad_norm_` for the parameters of the stack."""
        from ..ops.grad_clip import clip_grad_norm_

        return clip_grad_norm_(self.parameters(), max_norm, grad_scale)
