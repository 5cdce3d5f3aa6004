"""The norms before and after a block, fused with the block's gate and residual scale
(csrc/block_norm.hip):

    norm_before:  next = next_weight * rms(x)
    norm_after:   y    = resid + scale * sigmoid(gate) * weight * rms(h)
                  next = next_weight * rms(y)      (the following block's norm_before, same pass)

rms(z) = z / sqrt(mean(z^2) + eps) over the last dimension. float32, bfloat16 and float16 rows; the
parameters (vectors over the columns) are used, and their gradients summed, in float32; y is
rounded where it is returned, not on the way into next. GATModel(block_norm=True) wires a layer
stack with them. There is no CPU path."""
from __future__ import annotations

import torch
from torch import nn

from ._lib import host as _host


def norm_before(x, weight, eps: float = 1e-6):
    """weight * rms(x): the norm before a block. x: (..., D), weight: (D,), D <= 8192."""
    return _host.norm_before(x, weight, eps)


def norm_after(h, weight, *, resid=None, gate=None, scale=None, next_weight=None,
               eps: float = 1e-6):
    """y = resid + scale * sigmoid(gate) * weight * rms(h) for a block's output h (..., D), D <= 8192:
    the norm after the block, its gate, the residual scale and the residual. weight, scale: (D,);
    gate: (D,), a parameter, or of h's shape and dtype; resid of h's. Returns y, or with next_weight
    (D,) the pair (y, next_weight * rms(y)): the norm before the next block in the same pass. Once
    differentiable in every tensor, the same bits every time."""
    return _host.norm_after(h, weight, resid, gate, scale, next_weight, eps)


class BlockNorm(nn.Module):
    """The parameters of norm_after for one block of `features` columns: weight, a residual scale, a
    gate per column (gate=True) and the next block's norm (following=True)."""

    def __init__(self, features, gate=True, following=True, scale_init=1.0, eps=1e-6):
        super().__init__()
        self.features, self.eps, self.scale_init = features, eps, scale_init
        self.weight = nn.Parameter(torch.empty(features))
        self.scale = nn.Parameter(torch.empty(features))
        for name, wanted in (("gate", gate), ("next_weight", following)):
            self.register_parameter(name,
                                    nn.Parameter(torch.empty(features)) if wanted else None)
        self.reset_parameters()

    def reset_parameters(self):
        nn.init.ones_(self.weight)
        nn.init.constant_(self.scale, self.scale_init)
        if self.gate is not None:
            nn.init.zeros_(self.gate)
        if self.next_weight is not None:
            nn.init.ones_(self.next_weight)

    def forward(self, h, resid=None, gate=None):
        """y, or (y, next) with following; gate: one of h's shape instead of the parameter."""
        return norm_after(h, self.weight, resid=resid, gate=self.gate if gate is None else gate,
                          scale=self.scale, next_weight=self.next_weight, eps=self.eps)

    def extra_repr(self) -> str:
        return f"{self.features}, eps={self.eps}"
