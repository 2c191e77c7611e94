"""Block decoding of the Dream-shaped model with full attention over a paged cache.

The dense counterpart of the routed model (``dream_forward.py``) as a server
would run it: the layers' projections and MLP as there, q and k rotated and k
and v put into their pages in one launch (``paged_append``), attention over
the sequence's pages (``paged_attention``: a prompt's thousands of rows, a
block's 32 and a single token's one alike), and candidates that hold their
prompt's pages in common.

A denoising loop::

    dec = PagedDream(DreamForward(cfg), pages=4096, sequences=8, max_len=16384)
    seq, cands = dec.cache.seqs(0), dec.cache.seqs(1, 2, 3, 4)
    dec.prefill(seq, prompt)                                   # [1, L] token ids
    dec.fork(seq, cands)                                       # the prompt's pages, held in common
    at = dec.cache.lengths[1:5].clone()                        # where the blocks begin
    dec.cache.extend(cands, 32)                                # room for a block each
    for _ in range(steps):
        logits = dec.step(cands, block, start=at)              # [4, 32] ids: rewrites the block's keys and values
        block = choose(logits, block)
    dec.cache.free(losers)

With ``start`` given, a block whose ``extend`` was refused (no free pages, too
long) has no place and is not written; without it the last tokens that the
sequence does have would be.
"""

from __future__ import annotations

import torch

from .dream_forward import DreamForward
from .paged_cache import PagedKVCache


class PagedDream:
    """``model``'s weights (:class:`DreamForward`, or :class:`DreamInt8` for
    dense layers in 8 bits) with full attention and a cache of ``pages`` pages
    for all layers."""

    def __init__(self, model: DreamForward, *, pages: int, sequences: int, max_len: int, page_size: int = 64):
        c = model.cfg
        self.model = model
        self.cache = PagedKVCache(c.layers, pages, c.kv_heads, c.head_dim, sequences=sequences, max_len=max_len,
                                  page_size=page_size, device=model.embed.device)

    @torch.inference_mode()
    def step(self, seqs, ids, *, start=None, position_ids=None, key_valid=None, causal: bool = False,
             logits: bool = True):
        """Runs the tokens ``ids [B, S]`` of the sequences ``seqs`` at the cache
        positions from ``start`` on (default: each sequence's last S, which
        :meth:`PagedKVCache.extend` has made room for), writing their keys and
        values over what was there, and returns their logits (or the final
        hidden states).  Every token sees its whole sequence, or with
        ``causal`` (last positions only) the tokens up to itself."""
        m, c = self.model, self.model.cfg
        b, s = ids.shape
        x = m.begin(m.embed[ids])
        for idx in range(c.layers):
            q, k, v, _, x = m.enter(idx, x)
            q = self.cache.append(idx, seqs, k, v, q=q, start=start, position_ids=position_ids, inv_freq=m.inv_freq,
                                  attention_factor=m.attention_factor)
            o = self.cache.attend(idx, seqs, q, causal=causal, key_valid=key_valid)
            x = m.leave(idx, o.reshape(b, s, c.q_heads * c.head_dim), x)
        return m.end(x, logits)

    def prefill(self, seqs, ids, **kw):
        """The tokens ``ids [B, S]`` appended to the sequences: room for them,
        then :meth:`step` from where they ended before.  Without that room
        nothing is written, and :meth:`PagedKVCache.check` says why."""
        lengths = self.cache.lengths
        rows = seqs.clamp(0, lengths.shape[0] - 1)        # a number out of range is reported, not followed
        kw.setdefault("start", lengths.index_select(0, rows))
        self.cache.extend(seqs, ids.shape[1])
        return self.step(seqs, ids, **kw)

    def fork(self, src, dst, share=None) -> None:
        """Candidates: each of ``dst`` continues ``src`` (one sequence for all,
        or one each) and may rewrite what lies past ``share`` tokens."""
        if src.shape[0] == 1 and dst.shape[0] > 1:
            src = src.expand(dst.shape[0])
        if share is not None and share.shape[0] == 1 and dst.shape[0] > 1:
            share = share.expand(dst.shape[0])
        self.cache.fork(src, dst, share)


__all__ = ["PagedDream"]
