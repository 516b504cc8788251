"""``MXLoRALinear``: ``LoRALinear`` (``torchtune/modules/peft/lora.py:27-147``) over a frozen mxfp4 weight.

The input is quantised to mxfp8 once; base product and adapter read it, and it is all that is kept of the input for the
backward pass (8.25 bits per element).  Layers that read the same input share it, as long as their ranks add up to at most 64:
``lora_linear_group``.  Adapters and bias are bfloat16 in the forward pass (build the layer with that default dtype, or move it there).
"""
from __future__ import annotations

from typing import List

import torch
from torch import nn

from ...mx import linear_mx, lora_linear_mx
from ..low_precision.mx_linear import MXWeight
from ._adapter_base import _lora_a_init_params, _lora_b_init_params

MAX_RANK = 64  # of a layer, and of all the members of a group together


class MXLoRALinear(MXWeight):
    """Args:
        in_dim (int), out_dim (int): multiples of 64
        rank (int): rank of the adapter, a multiple of 8 up to 64
        alpha (float): adapter scaling numerator
        dropout (float): dropout on the adapter's input. Where it is active the adapter reads the unrounded input and autograd
            keeps it. Default 0.0
        use_bias (bool): whether the base linear has a bias. Default False

    Raises:
        ValueError: if a dimension or the rank is not supported
    """

    def __init__(self, in_dim: int, out_dim: int, rank: int, alpha: float, dropout: float = 0.0, use_bias: bool = False):
        super().__init__()
        if in_dim % 64 or out_dim % 64 or in_dim <= 0 or out_dim <= 0:
            raise ValueError(f"MXLoRALinear: in_dim and out_dim must be multiples of 64, got {in_dim} and {out_dim}")
        if rank % 8 or not 0 < rank <= MAX_RANK:
            raise ValueError(f"MXLoRALinear: the rank must be a multiple of 8 up to {MAX_RANK}, got {rank}")
        self.in_dim, self.out_dim, self.rank, self.alpha, self.use_bias = in_dim, out_dim, rank, alpha, use_bias
        self.disabled = False  # True: behave as the frozen base layer alone
        self.merged = False
        dense = nn.Linear(in_dim, out_dim, bias=use_bias)
        self._register_mx_weight(dense.weight)
        self.register_parameter("bias", nn.Parameter(dense.bias.detach()) if use_bias else None)
        self.dropout = nn.Dropout(p=dropout) if dropout > 0.0 else nn.Identity()
        self.lora_a = nn.Linear(in_dim, rank, bias=False)
        self.lora_b = nn.Linear(rank, out_dim, bias=False)
        self.initialize_parameters()

    def initialize_parameters(self):
        _lora_a_init_params(self.lora_a)
        _lora_b_init_params(self.lora_b)

    def adapter_params(self) -> List[str]:
        """Names of this module's adapter parameters."""
        return ["lora_a.weight", "lora_b.weight"]

    def _drops(self) -> bool:
        return self.training and isinstance(self.dropout, nn.Dropout) and self.dropout.p > 0.0

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """x ``(..., in_dim)`` -> ``(..., out_dim)``"""
        if self.disabled:
            return linear_mx(x, self.mx_weight, self.bias)
        if self._drops():
            return linear_mx(x, self.mx_weight, self.bias) + self.alpha / self.rank * self.lora_b(self.lora_a(self.dropout(x)))
        return mx_lora_group(x, (self,))[0]


def mx_group_applies(layers) -> bool:
    """True when these layers, which share an input, can run as one call."""
    return (1 <= len(layers) <= 4 and all(type(l) is MXLoRALinear and not l.disabled and not l._drops() and l.in_dim == layers[0].in_dim for l in layers)
            and sum(l.rank for l in layers) <= MAX_RANK)


def mx_lora_group(x: torch.Tensor, layers):
    return lora_linear_mx(x, [l.mx_weight for l in layers], [l.lora_a.weight for l in layers], [l.lora_b.weight for l in layers],
                          [l.alpha / l.rank for l in layers], [l.bias for l in layers])
