"""Rotary positions for any head layout, type and stride.

``rope_fp32`` holds the reference's rotary drop-ins (rotate-half, whole heads
of 128 bf16 dims, contiguous).  ``rotary_embedding`` is the general operator:
rotate-half or interleaved pairs, the first part of a head or all of it,
bf16, fp16 or fp32, views of a fused projection as they are, and its gradient.
"""

from __future__ import annotations

import torch

from . import _lib
from .rope_fp32 import yarn_inv_freq

def rotary_inv_freq(dim: int, base: float = 1.0e6, *, scaling: str = "none", factor: float = 1.0,
                    orig_max_pos: int = 2048, device=None):
    """Inverse frequencies ``[dim/2]`` (fp32) of ``dim`` rotated dims, and the
    attention factor, for a context ``factor`` times the trained one.

    ``scaling``: ``"none"``; ``"linear"`` divides every frequency by
    ``factor``; ``"ntk"`` raises the base to ``base * factor ** (dim / (dim -
    2))``, which keeps the fastest frequency and divides the slowest by
    ``factor``; ``"yarn"`` is :func:`yarn_inv_freq`."""
    if dim < 2 or dim % 2:
        raise ValueError(f"the rotated dims must be even and positive, got {dim}")
    if not factor > 0 or not base > 0:
        raise ValueError("base and factor must be positive")
    if scaling == "yarn":
        return yarn_inv_freq(dim, base, factor, orig_max_pos, device=device)
    if scaling == "ntk":
        if dim == 2:
            raise ValueError("ntk scaling needs more than two rotated dims")
        base = base * factor ** (dim / (dim - 2))
    elif scaling not in ("none", "linear"):
        raise ValueError(f"unknown scaling {scaling!r}")
    inv = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if scaling == "linear":
        inv = inv / factor
    return inv.to(dtype=torch.float32, device=device), 1.0


def rotary_embedding(q: torch.Tensor, k: torch.Tensor | None, position_ids: torch.Tensor, inv_freq: torch.Tensor,
                     attention_factor: float = 1.0, *, layout: str = "half"):
    """Rotary positions of ``q [B, L, Hq, D]`` and ``k [B, L, Hk, D]`` (or
    None), bf16, fp16 or fp32: ``(q', k')``, contiguous, of the same type.

    The first ``2 n`` dims of each head turn, ``n = len(inv_freq)``; ``layout``
    ``"half"`` pairs dims ``(i, i + n)``, ``"interleaved"`` ``(2i, 2i + 1)``;
    the other dims pass through.  The angle is the fp32 product ``position *
    inv_freq`` and cos and sin are times ``attention_factor``, as in
    :func:`yarn_rope_qk`; fp32 arithmetic, one rounding.  Any batch, token and
    head strides.  Records the gradient of q and k where one is wanted;
    a gradient of ``inv_freq`` and forward-mode tangents are refused."""
    return _lib.ext().rotary(q, k, position_ids, inv_freq, attention_factor, layout)
