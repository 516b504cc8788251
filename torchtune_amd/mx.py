"""Microscaled (MX) tensors and the linears that multiply them on gfx950's block-scaled matrix instructions.

An :class:`MXTensor` holds blocks of 32 consecutive elements of its last dimension under one power-of-two scale: ``mxfp4``
(4.25 bits per element) for weights and inputs, ``mxfp8`` (8.25 bits) for inputs.  :func:`to_mx` makes one,
``MXTensor.to(dtype)`` reads it back, :func:`linear_mx` multiplies an input, quantised on its way in, with a frozen mxfp4
weight, and :func:`lora_linear_mx` is the training form with low-rank adapters, which keeps its input for the backward pass
in 8 bits.  They stand beside ``to_nf4`` / ``linear_nf4`` / ``LoRALinear``: four bits per weight as well, but a format that
the matrix cores multiply without expanding it.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import ops

FORMATS = ("mxfp4", "mxfp8")
BLOCK = 32


def _check_format(format: str, what: str) -> str:
    if format not in FORMATS:
        raise ValueError(f"{what}: unknown format {format!r} (one of {', '.join(FORMATS)})")
    return format


class MXTensor:
    """A tensor in microscaled blocks.

    Args:
        codes (torch.Tensor): uint8; ``[..., K / 2]`` for mxfp4 (element ``2 i`` in the low half of byte ``i``), ``[..., K]``
            for mxfp8 (e4m3)
        scales (torch.Tensor): uint8 ``[..., K / 32]``: a block's scale is ``2 ** (scale - 127)``; 255 marks a block of NaN
        dtype (torch.dtype): what ``.to()`` without a dtype gives back. Default bfloat16
        format (str): "mxfp4" or "mxfp8". Default "mxfp4"

    Raises:
        TypeError: if ``codes`` or ``scales`` is not uint8
        ValueError: if the two do not fit each other, live on different devices, or the format is unknown
    """

    __slots__ = ("codes", "scales", "dtype", "format", "shape")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16, format: str = "mxfp4"):
        _check_format(format, "MXTensor")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError(f"MXTensor: codes and scales must be uint8, got {codes.dtype} and {scales.dtype}")
        per_block = BLOCK // 2 if format == "mxfp4" else BLOCK
        if codes.dim() == 0 or codes.shape[:-1] != scales.shape[:-1] or codes.shape[-1] != per_block * scales.shape[-1]:
            raise ValueError(f"MXTensor: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not fit each other as {format}")
        if codes.device != scales.device:
            raise ValueError(f"MXTensor: codes on {codes.device}, scales on {scales.device}")
        self.codes, self.scales, self.dtype, self.format = codes, scales, dtype, format
        self.shape = torch.Size((*codes.shape[:-1], BLOCK * scales.shape[-1]))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def to(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The dense tensor, bfloat16 or float32 (default: ``self.dtype``)."""
        return ops.mx_dequantize(self.codes, self.scales, self.format, self.dtype if dtype is None else dtype)

    def __repr__(self) -> str:
        return f"MXTensor(shape={tuple(self.shape)}, format={self.format}, dtype={self.dtype}, device={self.device})"


def to_mx(tensor: torch.Tensor, format: str = "mxfp4") -> MXTensor:
    """``tensor`` (bfloat16 or float32, last dimension a multiple of 32) in microscaled blocks.

    The scale of a block is ``2 ** (floor(log2(largest magnitude)) - 2)`` for mxfp4 and ``- 8`` for mxfp8, at least 2^-127;
    elements are rounded to nearest even and saturate at 6 and 448.  A block with an infinity or a NaN reads back as NaN.
    """
    _check_format(format, "to_mx")
    codes, scales = ops.mx_quantize(tensor, format)
    return MXTensor(codes, scales, tensor.dtype, format)


def _check_weight(weight: MXTensor, what: str) -> None:
    if not isinstance(weight, MXTensor) or weight.format != "mxfp4" or len(weight.shape) != 2:
        raise TypeError(f"{what}: the weight must be a 2-D mxfp4 MXTensor, got {weight!r}")


def _check_input(x: torch.Tensor, weight: MXTensor, what: str) -> None:
    n, k = weight.shape
    if x.dtype != torch.bfloat16:
        raise TypeError(f"{what}: expected a bfloat16 input, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] != k:
        raise RuntimeError(f"{what}: mat1 and mat2 shapes cannot be multiplied ({tuple(x.shape)} and {k}x{n})")
    if x.device != weight.device:
        raise RuntimeError(f"{what}: the input is on {x.device}, the weight on {weight.device}")


class _LinearMX(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, codes, scales, bias, activation: str):
        ctx.save_for_backward(codes, scales)
        ctx.x_shape = x.shape
        n, k = codes.shape[0], x.shape[-1]
        return ops.mx_linear(x.reshape(-1, k), codes, scales, activation, bias).view(*x.shape[:-1], n)

    @staticmethod
    def backward(ctx, gy):
        codes, scales = ctx.saved_tensors
        n = codes.shape[0]
        gx = gbias = None
        gy2 = gy.reshape(-1, n)
        if ctx.needs_input_grad[0]:
            gx = ops.mx_linear_dx(gy2, codes, scales).view(ctx.x_shape)
        if ctx.needs_input_grad[3]:
            gbias = gy2.sum(dim=0)
        return gx, None, None, gbias, None


def linear_mx(input: torch.Tensor, weight: MXTensor, bias: Optional[torch.Tensor] = None, activation: str = "mxfp8") -> torch.Tensor:
    """``input . weight^T (+ bias)`` with the input quantised to ``activation`` ("mxfp8" or "mxfp4") on its way in.

    ``input [..., K]`` bfloat16, ``weight [N, K]`` a frozen mxfp4 :class:`MXTensor`; fp32 sums, bfloat16 output.  The
    gradient of the input passes the rounding straight through (``gy . weight``); it takes N and K that are multiples of 64.
    """
    _check_format(activation, "linear_mx")
    _check_weight(weight, "linear_mx")
    _check_input(input, weight, "linear_mx")
    n, k = weight.shape
    if torch.is_grad_enabled() and input.requires_grad and (n % 64 or k % 64):
        raise ValueError(f"linear_mx: the gradient of the input needs a weight whose sides are multiples of 64, got {n} x {k}")
    if torch.is_grad_enabled() and (input.requires_grad or (bias is not None and bias.requires_grad)):
        return _LinearMX.apply(input, weight.codes, weight.scales, bias, activation)
    return ops.mx_linear(input.reshape(-1, k), weight.codes, weight.scales, activation, bias).view(*input.shape[:-1], n)


class _LoRALinearMX(torch.autograd.Function):
    """Inputs: x, the members' (scale, ...), n, then codes, scales, lora_a, lora_b and bias of each member in turn."""

    @staticmethod
    def forward(ctx, x, factors: Tuple[float, ...], *operands):
        n = len(factors)
        members = [ops.MxMember(*operands[5 * i:5 * i + 5], factors[i]) for i in range(n)]
        k = x.shape[-1]
        ys, codes, scales, h = ops.mx_lora_fwd(x.reshape(-1, k), members)
        ctx.save_for_backward(codes, scales, h, *operands)
        ctx.factors, ctx.x_shape = factors, x.shape
        return tuple(y.view(*x.shape[:-1], y.shape[-1]) for y in ys)

    @staticmethod
    def backward(ctx, *gys):
        codes, scales, h, *operands = ctx.saved_tensors
        n = len(ctx.factors)
        members = [ops.MxMember(*operands[5 * i:5 * i + 5], ctx.factors[i]) for i in range(n)]
        need = ctx.needs_input_grad
        gy2 = [gy.reshape(-1, m.codes.shape[0]) for gy, m in zip(gys, members)]
        gx, gas, gbs = ops.mx_lora_bwd(gy2, codes, scales, h, members, need_gx=need[0])
        out = [gx.view(ctx.x_shape) if need[0] else None, None]
        for i in range(n):
            needs = need[2 + 5 * i:7 + 5 * i]
            gbias = gy2[i].sum(dim=0) if members[i].bias is not None and needs[4] else None
            out += [None, None, gas[i] if needs[2] else None, gbs[i] if needs[3] else None, gbias]
        return tuple(out)


def lora_linear_mx(input: torch.Tensor, weights: Sequence[MXTensor], lora_a: Sequence[torch.Tensor], lora_b: Sequence[torch.Tensor],
                   scales: Sequence[float], biases: Optional[Sequence[Optional[torch.Tensor]]] = None) -> Tuple[torch.Tensor, ...]:
    """One or several adapter linears over frozen mxfp4 weights that read the same input:
    ``y_i = x^ . W_i^T (+ bias_i) + scales[i] * (x^ . lora_a[i]^T) . lora_b[i]^T`` with ``x^`` the input in mxfp8.

    ``x^`` is what is kept for the backward pass (8.25 bits per element, once for all members); the adapters' gradients are
    those of the products over it, the input's gradient passes the rounding straight through.  ``input [..., K]``,
    ``lora_a[i] [r, K]``, ``lora_b[i] [N, r]`` and biases bfloat16; N and K multiples of 64, ranks multiples of 8 that add
    up to at most 64, one to four members.
    """
    n = len(weights)
    biases = [None] * n if biases is None else list(biases)
    if not (1 <= n <= ops.GROUP_MAX and len(lora_a) == len(lora_b) == len(scales) == len(biases) == n):
        raise ValueError(f"lora_linear_mx: takes 1 to {ops.GROUP_MAX} weights and as many adapters, scales and biases, got "
                         f"{n}, {len(lora_a)}, {len(lora_b)}, {len(scales)}, {len(biases)}")
    total = 0
    for w, a, b, bias in zip(weights, lora_a, lora_b, biases):
        _check_weight(w, "lora_linear_mx")
        _check_input(input, w, "lora_linear_mx")
        (rows, k), r = w.shape, a.shape[0] if a.dim() == 2 else 0
        if r == 0 or r % 8 or a.shape[1] != k or tuple(b.shape) != (rows, r):
            raise ValueError(f"lora_linear_mx: lora_a {tuple(a.shape)} and lora_b {tuple(b.shape)} do not fit a weight of {rows} x {k} "
                             "with a rank that is a multiple of 8")
        if rows % 64 or k % 64:
            raise ValueError(f"lora_linear_mx: the weight's sides must be multiples of 64, got {rows} x {k}")
        if bias is not None and tuple(bias.shape) != (rows,):
            raise ValueError(f"lora_linear_mx: bias {tuple(bias.shape)} does not fit {rows} outputs")
        for t in (a, b, bias):
            if t is not None and t.dtype != torch.bfloat16:
                raise TypeError(f"lora_linear_mx: adapters and biases must be bfloat16, got {t.dtype}")
            if t is not None and t.device != input.device:
                raise RuntimeError(f"lora_linear_mx: the input is on {input.device}, an adapter or bias on {t.device}")
        total += r
    if total > 64:
        raise ValueError(f"lora_linear_mx: the members' ranks add up to {total}, at most 64 are supported")
    flat = []
    for w, a, b, bias in zip(weights, lora_a, lora_b, biases):
        flat += [w.codes, w.scales, a, b, bias]
    return _LoRALinearMX.apply(input, tuple(float(s) for s in scales), *flat)
