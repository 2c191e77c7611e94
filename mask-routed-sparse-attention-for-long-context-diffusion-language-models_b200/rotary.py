"""Rotary positions for any head layout, type and stride.

``rope_fp32`` holds the reference's rotary drop-ins (rotate-half, whole heads
of 128 bf16 dims, contiguous).  ``rotary_embedding`` is the general operator:
rotate-half or interleaved pairs, the first part of a head or all of it,
bf16, fp16 or fp32, views of a fused projection as they are, and its gradient.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .rope_fp32 import yarn_inv_freq

LAYOUTS = {"half": 0, "interleaved": 1}
DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}


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


def inner_contiguous(x: torch.Tensor) -> torch.Tensor:
    """``x`` as it is when its last dimension is contiguous, else a copy."""
    return x if x.stride()[-1] == 1 or x.shape[-1] == 1 else x.contiguous()


# The checks below are one condition on the path of a good call (a step of a
# few microseconds pays for each attribute it asks for); what exactly is wrong
# is found out where the condition fails.
def check_heads(x: torch.Tensor, name: str, like: torch.Tensor | None = None) -> None:
    """Raises unless x is a CUDA tensor (B, L, H, D) that fits ``like``."""
    if x.is_cuda and x.ndim == 4:
        if like is None:
            return
        if x.dtype is like.dtype and x.device == like.device:
            b, l, _, d = x.shape
            if (b, l, like.shape[2], d) == like.shape:
                return
    if not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if x.ndim != 4:
        raise ValueError(f"{name} must be (B, L, H, D)")
    raise ValueError(f"{name} must share type, device, (B, L) and D with the other heads")


def new_heads(b, l, h, d, dtype, device):
    """An uninitialised contiguous (B, L, H, D) tensor (``empty_strided``
    takes 1.5 us where ``empty``, with more to parse, takes 2.4 us)."""
    return torch.empty_strided((b, l, h, d), (l * h * d, h * d, d, 1), dtype=dtype, device=device)


def check_rotation(inv_freq, position_ids, batch, length, head_dim, layout, device):
    """``(inv_freq, pairs)``, the frequencies on the device in fp32."""
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {tuple(LAYOUTS)}, got {layout!r}")
    pairs = inv_freq.shape[0] if inv_freq.ndim == 1 else -1
    if not 1 <= pairs <= 128 or 2 * pairs > head_dim:
        raise ValueError(f"inv_freq must be [n] with 2 n <= D and n <= 128, got {tuple(inv_freq.shape)}, D={head_dim}")
    if position_ids is not None and (position_ids.shape != (batch, length) or position_ids.dtype is not torch.long or
                                     position_ids.device != device):
        raise ValueError("position_ids must be int64 (B, L) on the tensors' device")
    if inv_freq.dtype is not torch.float32 or inv_freq.device != device:
        inv_freq = inv_freq.to(device=device, dtype=torch.float32)
    return inv_freq if inv_freq.is_contiguous() else inv_freq.contiguous(), pairs


def _rotate(q, k, position_ids, inv_freq, pairs, factor, layout, inverse):
    qs = q.stride()
    if qs[3] != 1:
        q = inner_contiguous(q)
        qs = q.stride()
    b, l, hq, d = q.shape
    dtype, dev = q.dtype, q.device
    qo = new_heads(b, l, hq, d, dtype, dev)
    ko, hk, kp, kop, ks = None, 0, 0, 0, (0, 0, 0)
    if k is not None:
        ks = k.stride()
        if ks[3] != 1:
            k = inner_contiguous(k)
            ks = k.stride()
        hk = k.shape[2]
        ko = new_heads(b, l, hk, d, dtype, dev)
        kp, kop = k.data_ptr(), ko.data_ptr()
    args = _lib.ROTARY_ARGS.pack(q.data_ptr(), qo.data_ptr(), kp, kop, position_ids.data_ptr(), inv_freq.data_ptr(),
                                 qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], b, l, hq, hk, d, pairs,
                                 factor, DTYPES[dtype], LAYOUTS[layout], inverse)
    _lib.call_packed("mrsa_rotary", args, _lib.raw_stream(dev))
    return qo, ko


class _Rotary(torch.autograd.Function):
    """The gradient of a rotation is the rotation by minus the angle."""

    @staticmethod
    def forward(ctx, q, k, position_ids, inv_freq, pairs, factor, layout):
        ctx.save_for_backward(position_ids, inv_freq)
        ctx.rest = pairs, factor, layout
        return _rotate(q, k, position_ids, inv_freq, pairs, factor, layout, 0)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        pairs, factor, layout = ctx.rest
        dq, dk = _rotate(gq, gk, *ctx.saved_tensors, pairs, factor, layout, 1)
        return dq, dk, None, None, None, None, None


def rotary_embedding(q: torch.Tensor, k: torch.Tensor | None, position_ids: torch.Tensor, inv_freq: torch.Tensor,
                     attention_factor: float = 1.0, *, layout: str = "half"):
    """Rotary positions of ``q [B, L, Hq, D]`` and ``k [B, L, Hk, D]`` (or
    None), bf16, fp16 or fp32: ``(q', k')``, contiguous, of the same type.

    The first ``2 n`` dims of each head turn, ``n = len(inv_freq)``; ``layout``
    ``"half"`` pairs dims ``(i, i + n)``, ``"interleaved"`` ``(2i, 2i + 1)``;
    the other dims pass through.  The angle is the fp32 product ``position *
    inv_freq`` and cos and sin are times ``attention_factor``, as in
    :func:`yarn_rope_qk`; fp32 arithmetic, one rounding.  Any batch, token and
    head strides.  Records the gradient of q and k where one is wanted."""
    check_heads(q, "q")
    if q.dtype not in DTYPES:
        raise ValueError(f"q must be BF16, FP16 or FP32, got {q.dtype}")
    if k is not None:
        check_heads(k, "k", q)
    b, l, _, d = q.shape
    inv_freq, pairs = check_rotation(inv_freq, position_ids, b, l, d, layout, q.device)
    if layout == "interleaved" and d % 2:
        raise ValueError("the interleaved layout needs an even head dim")
    if not position_ids.is_contiguous():
        position_ids = position_ids.contiguous()
    factor = float(attention_factor)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, position_ids, inv_freq, pairs, factor, layout)
    return _rotate(q, k, position_ids, inv_freq, pairs, factor, layout, 0)
