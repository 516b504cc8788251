"""``FrozenMXLinear``: a linear whose weight is a frozen mxfp4 tensor, beside ``FrozenNF4Linear``
(``torchtune/modules/low_precision/nf4_linear.py:16-70``): the same constructor, forward through ``linear_mx``.

The codes and scales are buffers (``weight_codes`` uint8 ``[N, K / 2]``, ``weight_scales`` uint8 ``[N, K / 32]``).  A state
dict that has a dense ``weight`` for the module instead is quantised while it is loaded.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from ...mx import BLOCK, MXTensor, linear_mx, to_mx


def _pack(dense: torch.Tensor) -> MXTensor:
    """``dense`` as mxfp4, a float16 or float64 tensor by way of float32."""
    return to_mx(dense if dense.dtype in (torch.bfloat16, torch.float32) else dense.float(), "mxfp4")


class MXWeight(nn.Module):
    """Base of the modules over a frozen mxfp4 weight: its buffers, quantisation and loading."""

    def _register_mx_weight(self, dense: torch.Tensor) -> None:
        n, k = dense.shape
        if k % BLOCK:
            raise ValueError(f"{type(self).__name__}: in_dim must be a multiple of {BLOCK}, got {k}")
        if dense.device.type == "meta":
            codes, scales = (torch.empty(n, k // d, dtype=torch.uint8, device="meta") for d in (2, BLOCK))
        else:
            packed = _pack(dense.detach())
            codes, scales = packed.codes, packed.scales
        self.register_buffer("weight_codes", codes)
        self.register_buffer("weight_scales", scales)

    @property
    def mx_weight(self) -> MXTensor:
        return MXTensor(self.weight_codes, self.weight_scales, torch.bfloat16, "mxfp4")

    @torch.no_grad()
    def set_weight(self, dense: torch.Tensor) -> None:
        """Quantise ``dense [N, K]`` into the weight."""
        n, half = self.weight_codes.shape
        if tuple(dense.shape) != (n, 2 * half):
            raise ValueError(f"{type(self).__name__}: expected a weight of {n} x {2 * half}, got {tuple(dense.shape)}")
        packed = _pack(dense.to(self.weight_codes.device))
        self.weight_codes.copy_(packed.codes)
        self.weight_scales.copy_(packed.scales)

    def _quantise_for_loading(self, dense: torch.Tensor):
        """Codes and scales of a checkpoint's dense weight, on the module's device.  A module on the meta device has none to
        offer: its weight stays where the checkpoint's lies (``load_state_dict(..., assign=True)`` puts it there)."""
        here = self.weight_codes.device
        if here.type != "meta":
            packed = _pack(dense.to(here))
            return packed.codes, packed.scales
        if dense.device.type == "meta":
            return self.weight_codes, self.weight_scales
        packed = _pack(dense if dense.is_cuda else dense.to("cuda"))
        return packed.codes.to(dense.device), packed.scales.to(dense.device)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        dense = state_dict.get(prefix + "weight")
        if dense is None:
            super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
            return
        # load_state_dict hands its modules a copy of the caller's dictionary: the dense entry is replaced there alone
        state_dict.pop(prefix + "weight")
        if dense.dim() != 2 or tuple(dense.shape) != (self.weight_codes.shape[0], 2 * self.weight_codes.shape[1]):
            error_msgs.append(f"size mismatch for {prefix}weight: copying a param with shape {tuple(dense.shape)} from checkpoint, the "
                              f"shape in current model is {tuple(self.mx_weight.shape)}.")
            state_dict[prefix + "weight_codes"], state_dict[prefix + "weight_scales"] = self.weight_codes, self.weight_scales
        else:
            codes, scales = self._quantise_for_loading(dense.detach())
            state_dict[prefix + "weight_codes"], state_dict[prefix + "weight_scales"] = codes, scales
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)


class FrozenMXLinear(MXWeight):
    """Args:
        in_dim (int): input dimension, a multiple of 32 (64, and ``out_dim`` too, where gradients pass through)
        out_dim (int): output dimension
        bias (bool): a frozen bfloat16 bias. Default False
        device, dtype: of the dense weight that is initialised and quantised
        activation (str): format the input is quantised to on its way in, "mxfp8" or "mxfp4". Default "mxfp8"

    Raises:
        ValueError: if ``in_dim`` is no multiple of 32 or ``activation`` is unknown
    """

    def __init__(self, in_dim: int, out_dim: int, bias: bool = False, device: Optional[torch.device] = None,
                 dtype: Optional[torch.dtype] = None, activation: str = "mxfp8"):
        super().__init__()
        if activation not in ("mxfp8", "mxfp4"):
            raise ValueError(f"FrozenMXLinear: unknown format {activation!r} (one of mxfp4, mxfp8)")
        self.in_features, self.out_features, self.activation = in_dim, out_dim, activation
        dense = nn.Linear(in_dim, out_dim, bias=bias, device=device, dtype=dtype)
        self._register_mx_weight(dense.weight)
        self.register_parameter("bias", nn.Parameter(dense.bias.detach().to(torch.bfloat16), requires_grad=False) if bias else None)

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return linear_mx(input, self.mx_weight, self.bias, self.activation)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, activation={self.activation}"
