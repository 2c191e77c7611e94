"""The Dream-shaped model with its dense layers in 8-bit integers.

Weights are quantized once, a scale per output channel; activations as they
come, a scale per token.  q, k and v are one product, the norms hand their rows
over in 8 bits, and the residual's addition is part of the norm that follows,
so a layer is::

    add_rms_norm_int8 -> linear_int8 (q, k, v) -> attention -> quantize_int8 -> linear_int8 (o_proj)
    add_rms_norm_int8 -> swiglu_int8 -> quantize_int8 -> linear_int8 (down)

Attention, embeddings, norms' weights and the residual stream stay bf16; a
route layer's Q-Cal reads the normed input in bf16, so there the norm and its
quantization are two steps.
"""

from __future__ import annotations

import torch

from .dense import add_rms_norm
from .dream_forward import DreamForward
from .int8 import add_rms_norm_int8, linear_int8, quantize_int8, swiglu_int8


class DreamInt8(DreamForward):
    """``model`` with 8-bit dense layers; its other parameters are shared, and
    its own dense weights are not held."""

    def __init__(self, model: DreamForward):
        self.cfg = model.cfg
        self.embed, self.role, self.final_norm = model.embed, model.role, model.final_norm
        self.inv_freq, self.attention_factor = model.inv_freq, model.attention_factor
        self.lm_head = quantize_int8(model.lm_head)
        self.layers = []
        for lay in model.layers:
            new = {k: lay[k] for k in ("in_norm", "post_norm", "route") if k in lay}
            new["wqkv"] = quantize_int8(torch.cat((lay["wq"], lay["wk"], lay["wv"])))
            new["bqkv"] = torch.cat((lay["bq"], lay["bk"], lay["bv"]))
            for k in ("wo", "wgu", "wd"):
                new[k] = quantize_int8(lay[k])
            self.layers.append(new)

    def gate_up(self, idx):
        """The gate and up weights ``[F, H]`` that layer ``idx``'s whole numbers stand for, in fp32."""
        q, scale = self.layers[idx]["wgu"]
        blocks = (q.float() * scale[:, None]).view(self.cfg.ffn // 128, 2, 128, self.cfg.hidden)
        return blocks[:, 0].reshape(self.cfg.ffn, self.cfg.hidden), blocks[:, 1].reshape(self.cfg.ffn, self.cfg.hidden)

    def project(self, idx, h):
        return self._split(idx, *quantize_int8(h))

    def _split(self, idx, q8, scale):
        c, lay = self.cfg, self.layers[idx]
        qkv = linear_int8(q8, scale, *lay["wqkv"], lay["bqkv"]).view(*q8.shape[:2], -1, c.head_dim)
        return torch.split(qkv, (c.q_heads, c.kv_heads, c.kv_heads), dim=2)

    # The stream is a pair: what the last dense layer adds, and what it adds to.
    def begin(self, x):
        return x, None

    def stream(self, x):
        return x[0] if x[1] is None else x[0] + x[1]

    def enter(self, idx, x):
        lay, h = self.layers[idx], None
        if "route" in lay:
            h, x = add_rms_norm(*x, lay["in_norm"], self.cfg.rms_eps)
            q, k, v = self.project(idx, h)
        else:
            q8, scale, x = add_rms_norm_int8(*x, lay["in_norm"], self.cfg.rms_eps)
            q, k, v = self._split(idx, q8, scale)
        return q, k, v, h, x

    def layer(self, idx, x, position_ids, key_valid):
        q, k, v, h, x = self.enter(idx, x)
        return self.leave(idx, self.attend(idx, q, k, v, h, position_ids, key_valid), x)

    def leave(self, idx, o, x):
        lay = self.layers[idx]
        delta = linear_int8(*quantize_int8(o), *lay["wo"])
        q8, scale, x = add_rms_norm_int8(delta, x, lay["post_norm"], self.cfg.rms_eps)
        return linear_int8(*quantize_int8(swiglu_int8(q8, scale, *lay["wgu"])), *lay["wd"]), x

    def end(self, x, logits: bool = True):
        if not logits:
            return add_rms_norm(*x, self.final_norm, self.cfg.rms_eps)[0]
        q8, scale, _ = add_rms_norm_int8(*x, self.final_norm, self.cfg.rms_eps)
        return linear_int8(q8, scale, *self.lm_head)


__all__ = ["DreamInt8"]
