"""RMSNorm, rotary embedding, the SwiGLU gate, the chunk cross entropy and token log probabilities as single-pass HIP kernels
with autograd.

These are the memory-bound neighbours of the quantized linears inside a decoder layer.  The reference runs each as
a chain of eager kernels: ``RMSNorm`` (``torchtune/modules/rms_norm.py:11-41``), ``Llama3ScaledRoPE.forward``
(``torchtune/models/llama3_1/_position_embeddings.py:128-190``), ``FeedForward.forward``
(``torchtune/modules/feed_forward.py:50-53``).  Same arguments and results (to floating-point tolerance); bf16
tensors on the GPU only (``qk_norm_rope`` and ``token_logprobs``: float32 too), anything else raises.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence

import torch
from torch import nn

from .. import _host, ops


def rms_norm(x: torch.Tensor, scale: torch.Tensor, eps: float) -> torch.Tensor:
    """``bf16(x * rsqrt(mean(x^2) + eps)) * scale`` over the last dimension, computed in fp32."""
    return _host.call("rms_norm", x, scale, eps)


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, norm: "RMSNorm"):
    """``h = x + residual; return h, norm(h)``: the residual stream's addition and the norm of the next sub-block
    (``torchtune/modules/transformer.py:129-141``) as one pass forward and one backward; same bits as the separate ops."""
    return _host.call("add_rms_norm", x, residual, norm.scale, norm.eps)


class RMSNorm(nn.Module):
    """Root-mean-square normalisation computed in fp32: ``bf16(x * rsqrt(mean(x^2) + eps)) * scale``.

    Args:
        dim (int): embedding size
        eps (float): added to the mean square. Default: 1e-6
    """

    def __init__(self, dim: int, eps: float = 1e-6) -> None:
        super().__init__()
        self.normalized_shape = (dim,)
        self.eps = eps
        self.scale = nn.Parameter(torch.ones(dim))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return rms_norm(x, self.scale, self.eps)


class _RopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, cache):
        ctx.save_for_backward(cache)
        return ops.rope(x, cache, inverse=False)

    @staticmethod
    def backward(ctx, gy):
        (cache,) = ctx.saved_tensors
        return ops.rope(gy, cache, inverse=True), None


def apply_rope(x: torch.Tensor, cache: torch.Tensor) -> torch.Tensor:
    """Rotate consecutive pairs of ``x [b, s, n_h, h_d]`` by the angles in ``cache [s, h_d/2, 2]`` (cos, sin), fp32 math."""
    return _RopeFn.apply(x, cache)


def qkv_rope_repeat(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor):
    """What lies between the q / k / v projections and the attention (``torchtune/modules/attention.py:255-290``) as one
    kernel per direction: ``apply_rope(q)``, ``repeat_kv(apply_rope(k), rep)``, ``repeat_kv(v, rep)`` with
    ``rep = n_h // n_kv``, bit for bit."""
    return _host.call("qkv_rope_repeat", q, k, v, cache)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, cache: torch.Tensor, q_scale: Optional[torch.Tensor] = None,
                 k_scale: Optional[torch.Tensor] = None, *, eps: float = 1e-6, positions: Optional[torch.Tensor] = None,
                 sections: Optional[Sequence[int]] = None, interleaved: bool = True):
    """Norm of every query and key head, then its rotation, one pass forward and one backward, in fp32 and rounded once: for models that
    norm before they rotate.  (With a scale that differs within a pair the other order is another function; rotate with
    :func:`apply_rope` and norm after it for models of that kind.)

    Args:
        q, k (torch.Tensor): ``[b, s, n_h, h_d]`` and ``[b, s, n_kv, h_d]``, bfloat16 or float32, ``h_d`` a multiple of 16 up to 512.
            Views of one projection's output are read where they are.
        cache (torch.Tensor): float32 ``[positions, h_d / 2, 2]``, cosine and sine of every position and frequency
        q_scale, k_scale (Optional[torch.Tensor]): ``[h_d]``, of the type of ``q``: ``x / sqrt(mean(x^2) + eps) * scale`` per head.
            Default: no norm
        eps (float): added to the mean square
        positions (Optional[torch.Tensor]): row of ``cache`` for each token, ``[b, s]`` or what broadcasts to it; with ``sections``
            ``[axes, b, s]``.  Default: 0, 1, .. in every sequence.  A position that is not in ``cache`` gives NaN.
        sections (Optional[Sequence[int]]): with positions of two to four axes (time, height, width): how many consecutive
            frequencies follow each; they add up to ``h_d / 2``
        interleaved (bool): frequency ``i`` turns elements ``2 i`` and ``2 i + 1``; else ``i`` and ``h_d / 2 + i``

    Returns:
        the two outputs, contiguous.  Differentiable once with respect to ``q``, ``k`` and the scales.
    """
    return _host.call("qk_norm_rope", q, k, cache, q_scale, k_scale, float(eps), positions, [] if sections is None else [int(n) for n in sections],
                      bool(interleaved))


class _RepeatKVFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rep: int):
        ctx.rep = rep
        return ops.repeat_kv(x, rep)

    @staticmethod
    def backward(ctx, gy):
        return ops.repeat_kv_bwd(gy, ctx.rep), None


def repeat_kv(x: torch.Tensor, rep: int) -> torch.Tensor:
    """``x.unsqueeze(3).expand(b, s, n_kv, rep, h_d).flatten(2, 3)`` for ``x`` ``[b, s, n_kv, h_d]``: the grouped-query
    expansion of key / value heads (``torchtune/modules/attention.py:284-290``) as one copy kernel, with the sum over the
    copies as its backward."""
    return _RepeatKVFn.apply(x, rep)


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` with the eager sequence's two bf16 roundings."""
    return _host.call("swiglu", gate, up)


class _CrossEntropySumFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target, ignore_index: int, scale: float):
        loss, grad = ops.cross_entropy_fwd_bwd(logits, target, ignore_index, scale)
        ctx.save_for_backward(grad)
        return loss.sum() * scale

    @staticmethod
    def backward(ctx, g):
        (grad,) = ctx.saved_tensors
        return grad.mul_(g.float().reshape(1)), None, None, None  # a 1-D fp32 factor: product in fp32, rounded to bf16 once


class _LinearCrossEntropySumFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index: int, scale: float):
        logits = torch.nn.functional.linear(hidden, weight)
        loss, grad = ops.cross_entropy_fwd_bwd(logits, target, ignore_index, scale)
        ctx.save_for_backward(grad, hidden, weight)
        return loss.sum() * scale

    @staticmethod
    def backward(ctx, g):
        grad, hidden, weight = ctx.saved_tensors
        gh = gw = None
        # the incoming scalar multiplies the small products, not the [rows, vocabulary] gradient of the logits
        if ctx.needs_input_grad[0]:
            gh = (grad @ weight).mul_(g.float().reshape(1))
        if ctx.needs_input_grad[1]:
            gw = (grad.t() @ hidden).mul_(g.float().reshape(1))
        return gh, gw, None, None, None


def linear_cross_entropy_sum(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                             scale: float = 1.0) -> torch.Tensor:
    """``scale * F.cross_entropy((hidden @ weight.T).float(), target, reduction="sum")`` for one chunk of rows: the
    vocabulary projection and the loss of the reference's ``LinearCrossEntropyLoss.compute_cross_entropy``
    (``torchtune/modules/loss/cross_entropy_loss.py:86-112``) as one autograd node, so that backward scales the
    ``[rows, dim]`` (and ``[vocabulary, dim]``) products by the incoming gradient instead of the logits' gradient."""
    return _LinearCrossEntropySumFn.apply(hidden, weight, target, ignore_index, scale)


def cross_entropy_sum(logits: torch.Tensor, target: torch.Tensor, ignore_index: int = -100, scale: float = 1.0) -> torch.Tensor:
    """``scale * F.cross_entropy(logits.float(), target, reduction="sum", ignore_index=ignore_index)`` for bf16 logits
    ``[rows, V]``: the per-chunk body of the reference's ``LinearCrossEntropyLoss``
    (``torchtune/modules/loss/cross_entropy_loss.py:86-112``).  The gradient w.r.t. the logits is produced in the same
    pass (pre-multiplied by ``scale``) and only rescaled by the incoming gradient in backward; call backward once."""
    return _CrossEntropySumFn.apply(logits, target, ignore_index, scale)


class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` returns; ``None`` where it was not asked for."""

    logprobs: torch.Tensor
    entropy: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0, entropy: bool = False, top: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of given tokens under ``softmax(logits / temperature)``, with the entropy and the most likely
    alternatives: what preference and policy losses and distillation are made of (in the reference, ``torchtune/rlhf/``, an eager
    log softmax and a gather) and what a sampler reports.  The logits are read once
    forward, and once more backward; no tensor of their size is kept beside them.

    Args:
        logits (torch.Tensor): ``[.., V]``, bfloat16 or float32; a shifted view such as ``logits[:, :-1]`` is read where it is
        tokens (torch.Tensor): int64, a token for each row ``[..]`` or several ``[.., n]``; the same one may occur twice.  The
            backward compares a row's tokens with each other: 256 of them cost little, thousands their square
        temperature (float): between 1e-6 and 1e6. Default: 1
        entropy (bool): also return ``-sum p log p`` of each row
        top (int): also return that many largest log probabilities, at most 64, with their tokens; of equal logits the lower
            token comes first.  Of a row with fewer than ``top`` tokens above ``-inf``, or with thousands of equal largest ones, each
            alternative costs about one more pass over the row
        ignore_index (int): a token that stands for none: its log probability is 0 and has no gradient.  Any other token
            outside the vocabulary gives NaN.

    Returns:
        :class:`TokenLogprobs`, float32 and int64.  ``logprobs`` and ``entropy`` are differentiable once with respect to the
        logits, ``top_logprobs`` is not (pass its tokens as ``tokens`` to train on them).  A row of nothing but ``-inf`` has log
        probabilities of ``-inf``, entropy 0 and no gradient; NaN or ``+inf`` in a row makes all of it NaN.
    """
    logprobs, ent, top_logprobs, top_tokens = _host.call("token_logprobs", logits, tokens, float(temperature), bool(entropy), int(top), int(ignore_index))
    return TokenLogprobs(logprobs, ent if entropy else None, top_logprobs if top else None, top_tokens if top else None)
