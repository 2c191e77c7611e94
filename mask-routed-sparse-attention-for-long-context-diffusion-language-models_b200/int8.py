"""Dense layers in 8-bit integers.

A row of values is held as whole numbers in [-127, 127] and one fp32 scale
(:func:`quantize_int8`): weights once, a scale per output channel, and
activations as they come, a scale per token.  :func:`linear_int8` and
:func:`swiglu_int8` multiply them on the tensor cores at twice the rate of bf16
and read half the bytes of the weights, which is what a block of few tokens
costs.  :func:`add_rms_norm_int8` gives the norm of a residual stream in that
form without a pass of its own::

    wq, ws = quantize_int8(weight)                      # [N, K], once
    q, scale, x = add_rms_norm_int8(delta, x, norm_weight, eps)
    y = linear_int8(q, scale, wq, ws, bias)

The products' sums are exact and their outputs rounded alike, so their rows do
not depend on how many a call has; nor do quantized rows.  The scales of
:func:`add_rms_norm_int8` do in their last bits, as :func:`add_rms_norm` says:
a sequence's values may differ by that from one batch to another.  Forward only: each operator raises under autograd rather than lose a
gradient.
"""

from __future__ import annotations

import torch

from . import _lib


def quantize_int8(x: torch.Tensor):
    """``(q, scale)``: each row (last dimension) of ``x`` (bf16, fp16 or fp32)
    as int8 whole numbers and an fp32 scale, ``scale = max|x| / 127`` and ``q``
    the whole number nearest ``x * (127 / max|x|)`` in 64 bits (the reciprocal of
    ``max|x|`` times 127, as torch divides), of two the even one.  Zeros have scale 0; a row with a NaN or an
    infinity has scale NaN, and so has what is computed from it.  ``q`` has
    ``x``'s shape, its rows on 16-byte boundaries."""
    return _lib.ext().quantize_int8(x)


def add_rms_norm_int8(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float):
    """``(q, scale, h)``: :func:`add_rms_norm` with its norm in 8 bits, as
    :func:`quantize_int8` gives it (of the norm in fp32, not rounded before;
    ``q`` is that of ``h * weight``, products of fp32 numbers rounded to fp32)."""
    return _lib.ext().add_rms_norm_int8(x, residual, weight, eps)


def linear_int8(q: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: torch.Tensor | None = None, *, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``sum_k q[..., k] * weight[n, k] * scale * weight_scale[n] + bias[n]``
    of int8 ``q [..., K]`` and ``weight [N, K]``, fp32 scales ``[...]`` and
    ``[N]``, and a bias ``[N]`` of any float type: exact sums, times the row's
    scale and then the channel's in fp32, rounded once to ``dtype`` (bf16, fp16
    or fp32).  K at most 131071.  Rows that do not start on 16-byte boundaries
    are copied first (those of :func:`quantize_int8` do)."""
    return _lib.ext().linear_int8(q, scale, weight, weight_scale, bias, dtype, False)


def swiglu_int8(q: torch.Tensor, scale: torch.Tensor, w_gate_up: torch.Tensor, w_scale: torch.Tensor, *,
                dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``silu(gate) * up`` of the two products with the interleaved weights of
    :func:`interleave_gate_up` (quantized after interleaving), in fp32, rounded
    once to ``dtype``."""
    return _lib.ext().linear_int8(q, scale, w_gate_up, w_scale, None, dtype, True)


__all__ = ["add_rms_norm_int8", "linear_int8", "quantize_int8", "swiglu_int8"]
