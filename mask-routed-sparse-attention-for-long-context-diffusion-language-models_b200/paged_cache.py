"""Pages of a key-value cache, and the attention that reads them.

The cache of all layers is one pool of pages; a sequence is a row of page
numbers.  Candidates of one prompt hold its pages in common
(:func:`page_fork`), a thinned prompt gives its gaps back
(:func:`page_compact`), and :func:`paged_append` rotates a step's q and k and
puts k and v into their pages in one launch.  Every operator works on the
device's own table: nothing waits for the GPU, and a call that cannot be
carried out says so in a status word (:meth:`PagedKVCache.check` reads it) and
leaves the table as it was (a fork without pages leaves its targets empty).

The operators take plain tensors, so that a server can keep its own
bookkeeping next to them:

* ``pool``: ``[layers, 2, pages, page_size, kv_heads, D]``, each page one
  contiguous block (``pool.transpose(3, 4)`` of a pool with the heads outside
  is one too);
* ``table``: int32 ``[sequences, max_pages]``, -1 where there is no page;
* ``lengths``: int32 ``[sequences]``, tokens;
* ``refcount``: int32 ``[pages]``, the sequences that hold each page;
* ``seqs`` and the like: int32 on the device, rows of the table.

New pages are the lowest free ones, in the order of the call's sequences and
then of their positions.  :class:`PagedKVCache` holds a set of them.
"""

from __future__ import annotations

import torch

from . import _lib

PAGE_SIZES = (16, 32, 64, 128, 256)

BAD_SEQUENCE, NO_PAGES, TOO_LONG, OUTSIDE, SHARED, CLASH = 1, 2, 4, 8, 16, 32
_STATUS = {BAD_SEQUENCE: "a sequence number is out of range or was given twice",
           NO_PAGES: "the pool has not enough free pages",
           TOO_LONG: "a sequence would outgrow its row of the table",
           OUTSIDE: "a token or a page number lies outside its sequence or the pool",
           SHARED: "a write to a page that several sequences hold",
           CLASH: "a page is copied to twice, or copied to and from, in one call"}


def page_free(table, lengths, refcount, seqs, *, status=None) -> None:
    """The sequences ``seqs`` give up their pages (rows -1, lengths 0).  A row
    that is out of range or comes twice: nothing is done, ``status`` says so."""
    _lib.ext().free(table, lengths, refcount, seqs, status)


def page_extend(table, lengths, refcount, seqs, tokens, *, page_size: int, status=None) -> None:
    """Sequence ``seqs[i]`` grows by ``tokens`` (one whole number, or int32
    ``[n]``) tokens, on new pages where its last one is full.  If one of them
    does not fit, none grows and ``status`` says why."""
    _lib.ext().extend(table, lengths, refcount, seqs, tokens, page_size, status)


def page_fork(pool, table, lengths, refcount, src, dst, share=None, *, status=None) -> None:
    """Sequence ``dst[i]`` gives up its pages and becomes a copy of ``src[i]``:
    the whole pages below ``share[i]`` tokens (int32 ``[n]``; None: the
    source's length) are held in common, the others are copied in every layer.
    ``dst`` are distinct and none is a source.  A sequence may write from
    ``share[i]`` on without touching its source, so a block that will be
    rewritten is given its own pages by ``share`` = where it begins.  If the
    pool does not hold the copies, every ``dst`` is left empty and ``status``
    says so."""
    _lib.ext().fork(pool, table, lengths, refcount, src, dst, share, status)


def page_compact(pool, table, lengths, refcount, seqs, keep, *, status=None) -> None:
    """Sequence ``seqs[i]`` keeps the tokens where ``keep[i]`` (bool ``[n,
    max_pages * page_size]``) is true, in order and in every layer.  The pages
    before its first dropped token stay as they are; the kept tokens after
    them move into new pages, and the old ones are given up (pages that other
    sequences hold too are never written).  If the pool does not hold the new
    pages, nothing changes and ``status`` says so."""
    _lib.ext().compact(pool, table, lengths, refcount, seqs, keep, status)


def page_copy(pool, src, dst, *, status=None) -> None:
    """Page ``src[i]`` copied to page ``dst[i]`` (int32 ``[n]``) in every
    layer; a page number out of range is skipped and ``status`` says so.  If a
    page is copied to twice, or both copied from and to (a page copied to
    itself stays as it is), nothing is copied and ``status`` says so."""
    _lib.ext().copy(pool, src, dst, status)


def paged_append(k_pages, v_pages, table, lengths, seqs, k, v, *, q=None, position_ids=None, inv_freq=None,
                 attention_factor: float = 1.0, layout: str = "half", start=None, refcount=None, status=None):
    """k and v ``[B, L, kv_heads, D]`` of the sequences ``seqs`` ``[B]`` into
    their pages of one layer (``k_pages``, ``v_pages`` ``[pages, page_size,
    kv_heads, D]``), at the cache positions from ``start[i]`` on (int32
    ``[B]``; None: the last L of each sequence), which the sequences must
    already have (:func:`page_extend`).

    With ``inv_freq`` q and k are turned first as in
    :func:`rotary_embedding`, at ``position_ids`` (None: the cache
    positions).  Returns q, turned, or None without one.  A token outside its
    sequence, or (with ``refcount``) on a page that several sequences hold, is
    not written, nor is a row of the batch that names tokens which an earlier
    row of it writes; ``status`` says so.  Forward only: it raises under
    autograd rather than return a q without its gradient."""
    return _lib.ext().append(k_pages, v_pages, table, lengths, seqs, k, v, q, position_ids, inv_freq, attention_factor,
                             layout, start, refcount, status)


def paged_attention(q, k_pages, v_pages, table, lengths, seqs, *, causal: bool = False, key_valid=None,
                    scale: float | None = None, return_lse: bool = False, status=None):
    """Attention of ``q [B, L, Hq, D]`` (bf16 or fp16, D 64 or 128) over the
    cached tokens of the sequences ``seqs`` ``[B]`` in one layer's pages, which
    hold the same type (fp32 pages can be appended to, but not attended to).

    The queries are a sequence's newest L tokens, whose keys and values the
    cache already holds: every query sees the whole sequence, as a block that
    is denoised does, or with ``causal`` the tokens up to its own position,
    ``length - L + i``.  ``key_valid`` (bool ``[B, max_pages * page_size]``)
    masks cached tokens; what masked tokens and unused slots hold does not
    matter.  Returns ``o [B, L, Hq, D]``, with ``return_lse`` also the
    natural-log LSE ``[B, L, Hq]`` in fp32; a query that sees no token gets
    zeros and -inf, one that sees a NaN or a score of +inf gets NaN in both.
    A weight of zero does not cancel a cached value that is not finite: with
    ``causal`` it may reach the queries before its token too.  ``scale``
    defaults to ``D ** -0.5``.  Forward only: it
    raises under autograd rather than return an output without a gradient."""
    return _lib.ext().attend(q, k_pages, v_pages, table, lengths, seqs, causal, key_valid, scale, return_lse, status)


class PagedKVCache:
    """A pool of pages for ``layers`` layers and the bookkeeping of at most
    ``sequences`` sequences of at most ``max_len`` tokens.  The methods are
    the module's operators on its tensors; sequence numbers are int32 tensors
    on the device (:meth:`seqs` makes one).  Pages start uninitialised: only
    tokens that were appended are ever read."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int, *, sequences: int, max_len: int,
                 page_size: int = 64, dtype=torch.bfloat16, device="cuda"):
        if min(layers, pages, kv_heads, head_dim, sequences, max_len) < 1:
            raise ValueError("every size of a cache must be positive")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        dev = torch.device(device)
        self.page_size = page_size
        self.pool = torch.empty(layers, 2, pages, page_size, kv_heads, head_dim, dtype=dtype, device=dev)
        self.table = torch.full((sequences, -(-max_len // page_size)), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=dev)
        self.refcount = torch.zeros(pages, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)

    def seqs(self, *numbers: int) -> torch.Tensor:
        """Sequence numbers on the cache's device."""
        return torch.tensor(numbers, dtype=torch.int32, device=self.table.device)

    def free(self, seqs) -> None:
        page_free(self.table, self.lengths, self.refcount, seqs, status=self.status)

    def extend(self, seqs, tokens) -> None:
        page_extend(self.table, self.lengths, self.refcount, seqs, tokens, page_size=self.page_size,
                    status=self.status)

    def fork(self, src, dst, share=None) -> None:
        page_fork(self.pool, self.table, self.lengths, self.refcount, src, dst, share, status=self.status)

    def compact(self, seqs, keep) -> None:
        page_compact(self.pool, self.table, self.lengths, self.refcount, seqs, keep, status=self.status)

    def append(self, layer: int, seqs, k, v, **kw):
        """:func:`paged_append` to one layer (``q``, ``inv_freq`` and the rest as there)."""
        return paged_append(self.pool[layer, 0], self.pool[layer, 1], self.table, self.lengths, seqs, k, v,
                            refcount=self.refcount, status=self.status, **kw)

    def attend(self, layer: int, seqs, q, **kw):
        """:func:`paged_attention` over one layer."""
        return paged_attention(q, self.pool[layer, 0], self.pool[layer, 1], self.table, self.lengths, seqs,
                               status=self.status, **kw)

    def check(self) -> None:
        """Waits for the device, clears the status word, and raises if a call
        since the last check could not be carried out."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            what = "; ".join(text for bit, text in _STATUS.items() if bits & bit)
            raise (RuntimeError if bits & NO_PAGES else ValueError)(f"paged cache: {what}")


__all__ = ["PAGE_SIZES", "PagedKVCache", "page_compact", "page_copy", "page_extend", "page_fork", "page_free",
           "paged_append", "paged_attention"]
