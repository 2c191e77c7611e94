"""Pages of a key-value cache, and the attention that reads them.

The cache of all layers is one pool of pages; a sequence is a row of page
numbers.  Candidates of one prompt hold its pages in common
(:func:`page_fork`), a thinned prompt gives its gaps back
(:func:`page_compact`), and :func:`paged_append` rotates a step's q and k and
puts k and v into their pages in one launch.  Every operator works on the
device's own table: nothing waits for the GPU, and a call that cannot be
carried out says so in a status word (:meth:`PagedKVCache.check` reads it).

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
from .rotary import DTYPES, LAYOUTS, check_heads, check_rotation, inner_contiguous, new_heads

PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_SEQS = 1024    # sequences per call of the page operators

BAD_SEQUENCE, NO_PAGES, TOO_LONG, OUTSIDE, SHARED = 1, 2, 4, 8, 16
_STATUS = {BAD_SEQUENCE: "a sequence number is out of range or was given twice",
           NO_PAGES: "the pool has not enough free pages",
           TOO_LONG: "a sequence would outgrow its row of the table",
           OUTSIDE: "a token or a page number lies outside its sequence or the pool",
           SHARED: "a write to a page that several sequences hold"}


def _ints(x: torch.Tensor, name: str, ndim: int, device=None) -> torch.Tensor:
    if x.dtype is not torch.int32 or x.ndim != ndim or not x.is_cuda:
        raise ValueError(f"{name} must be an int32 CUDA tensor with {ndim} dimension{'s' if ndim > 1 else ''}")
    if device is not None and x.device != device:
        raise ValueError(f"{name} must be on the table's device")
    return x if x.is_contiguous() else x.contiguous()


def _page_table(table, lengths, refcount, status, pages, page_size) -> bytes:
    """``mrsa_page_table``; the state tensors themselves are written, so they
    have to be contiguous."""
    dev, i32 = table.device, torch.int32
    if table.dtype is not i32 or table.ndim != 2 or not table.is_cuda or not table.is_contiguous():
        raise ValueError("table must be a contiguous int32 CUDA tensor [sequences, max_pages]")
    n, w = table.shape
    if lengths.dtype is not i32 or lengths.shape != (n,) or lengths.device != dev or not lengths.is_contiguous():
        raise ValueError("lengths must be contiguous int32 [sequences] on the table's device")
    rp = sp = 0
    if refcount is not None:
        if refcount.dtype is not i32 or refcount.ndim != 1 or refcount.device != dev or not refcount.is_contiguous():
            raise ValueError("refcount must be contiguous int32 [pages] on the table's device")
        if pages is None:
            pages = refcount.shape[0]
        elif refcount.shape[0] != pages:
            raise ValueError(f"refcount has {refcount.shape[0]} pages, the pool {pages}")
        rp = refcount.data_ptr()
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    if status is not None:
        if status.dtype is not i32 or status.numel() != 1 or status.device != dev:
            raise ValueError("status must be one int32 on the table's device")
        sp = status.data_ptr()
    return _lib.PAGE_TABLE.pack(table.data_ptr(), lengths.data_ptr(), rp, sp, n, w, pages, page_size)


def _page_pool(pool, device) -> bytes:
    """``mrsa_page_pool`` of ``[layers, 2, pages, page_size, heads, D]``."""
    if pool.ndim != 6 or pool.shape[1] != 2 or pool.device != device:
        raise ValueError("pool must be [layers, 2, pages, page_size, kv_heads, D] on the table's device")
    layers, _, _, ps, heads, d = pool.shape
    s, e = pool.stride(), pool.element_size()
    if s[5] != 1 or (s[3], s[4]) not in ((heads * d, d), (d, ps * d)):
        raise ValueError("each page of the pool must be one contiguous block, tokens or heads outside")
    return _lib.PAGE_POOL.pack(pool.data_ptr(), layers, s[0] * e, s[1] * e, s[2] * e, s[3] * e, s[4] * e, heads, d * e)


def _workspace(pt: bytes, n: int, device) -> tuple[torch.Tensor, int]:
    size = _lib.load().mrsa_page_workspace(pt, n)
    return torch.empty_strided((size,), (1,), dtype=torch.uint8, device=device), size


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """``x``, or a copy that begins on 16 bytes."""
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _count(x: torch.Tensor, name: str) -> int:
    n = x.shape[0]
    if n > MAX_SEQS:
        raise ValueError(f"{name}: at most {MAX_SEQS} sequences per call, got {n}")
    return n


def page_free(table, lengths, refcount, seqs, *, status=None) -> None:
    """The sequences ``seqs`` give up their pages (rows -1, lengths 0).  A row
    that is out of range or comes twice: nothing is done, ``status`` says so."""
    seqs = _ints(seqs, "seqs", 1, table.device)
    n = _count(seqs, "seqs")
    pt = _page_table(table, lengths, refcount, status, None, PAGE_SIZES[0])
    _lib.call_packed("mrsa_page_free", pt, seqs.data_ptr(), n, _lib.raw_stream(table.device))


def page_extend(table, lengths, refcount, seqs, tokens, *, page_size: int, status=None) -> None:
    """Sequence ``seqs[i]`` grows by ``tokens`` (one whole number, or int32
    ``[n]``) tokens, on new pages where its last one is full.  If one of them
    does not fit, none grows and ``status`` says why."""
    dev = table.device
    seqs = _ints(seqs, "seqs", 1, dev)
    n = _count(seqs, "seqs")
    more, each = 0, None
    if torch.is_tensor(tokens):
        each = _ints(tokens, "tokens", 1, dev)
        if each.shape != seqs.shape:
            raise ValueError("tokens must hold one number per sequence")
    else:
        more = int(tokens)
        if more < 0:
            raise ValueError("a sequence cannot grow by a negative number of tokens")
    pt = _page_table(table, lengths, refcount, status, None, page_size)
    if n == 0:
        return
    ws, size = _workspace(pt, n, dev)
    _lib.call_packed("mrsa_page_extend", pt, seqs.data_ptr(), 0 if each is None else each.data_ptr(), more, n, ws.data_ptr(),
              size, _lib.raw_stream(dev))


def page_fork(pool, table, lengths, refcount, src, dst, share=None, *, status=None) -> None:
    """Sequence ``dst[i]`` gives up its pages and becomes a copy of ``src[i]``:
    the whole pages below ``share[i]`` tokens (int32 ``[n]``; None: the
    source's length) are held in common, the others are copied in every layer.
    ``dst`` are distinct and none is a source.  A sequence may write from
    ``share[i]`` on without touching its source, so a block that will be
    rewritten is given its own pages by ``share`` = where it begins.  If the
    pool does not hold the copies, every ``dst`` is left empty and ``status``
    says so."""
    dev = table.device
    src, dst = _ints(src, "src", 1, dev), _ints(dst, "dst", 1, dev)
    n = _count(dst, "dst")
    sp = 0
    if share is not None:
        share = _ints(share, "share", 1, dev)
        sp = share.data_ptr()
    if src.shape != dst.shape or (share is not None and share.shape != dst.shape):
        raise ValueError("src, dst and share must have one entry per fork")
    pp = _page_pool(pool, dev)
    pt = _page_table(table, lengths, refcount, status, pool.shape[2], pool.shape[3])
    if n == 0:
        return
    ws, size = _workspace(pt, n, dev)
    _lib.call_packed("mrsa_page_fork", pt, pp, src.data_ptr(), dst.data_ptr(), sp, n, ws.data_ptr(), size,
              _lib.raw_stream(dev))


def page_compact(pool, table, lengths, refcount, seqs, keep, *, status=None) -> None:
    """Sequence ``seqs[i]`` keeps the tokens where ``keep[i]`` (bool ``[n,
    max_pages * page_size]``) is true, in order and in every layer.  The pages
    before its first dropped token stay as they are; the kept tokens after
    them move into new pages, and the old ones are given up (pages that other
    sequences hold too are never written).  If the pool does not hold the new
    pages, nothing changes and ``status`` says so."""
    dev = table.device
    seqs = _ints(seqs, "seqs", 1, dev)
    n = _count(seqs, "seqs")
    pp = _page_pool(pool, dev)
    width = table.shape[1] * pool.shape[3]
    if keep.dtype != torch.bool or keep.shape != (n, width) or keep.device != dev:
        raise ValueError(f"keep must be bool {(n, width)} on the table's device")
    pt = _page_table(table, lengths, refcount, status, pool.shape[2], pool.shape[3])
    if n == 0:
        return
    keep = _aligned(keep.contiguous())
    ws, size = _workspace(pt, n, dev)
    _lib.call_packed("mrsa_page_compact", pt, pp, seqs.data_ptr(), keep.data_ptr(), n, ws.data_ptr(), size,
              _lib.raw_stream(dev))


def page_copy(pool, src, dst, *, status=None) -> None:
    """Page ``src[i]`` copied to page ``dst[i]`` (int32 ``[n]``) in every
    layer; a page number out of range is skipped and ``status`` says so."""
    dev = pool.device
    src, dst = _ints(src, "src", 1, dev), _ints(dst, "dst", 1, dev)
    if src.shape != dst.shape:
        raise ValueError("src and dst must have one entry per page")
    n = src.shape[0]
    if n > pool.shape[2]:
        raise ValueError(f"{n} copies into {pool.shape[2]} pages")
    pp = _page_pool(pool, dev)
    if n == 0:
        return
    # the copy needs no table: the struct's is any valid pointer that is not read
    sp = 0 if status is None else _ints(status.reshape(1), "status", 1, dev).data_ptr()
    pt = _lib.PAGE_TABLE.pack(src.data_ptr(), src.data_ptr(), 0, sp, 1, 1, pool.shape[2], pool.shape[3])
    _lib.call_packed("mrsa_page_copy", pt, pp, src.data_ptr(), dst.data_ptr(), n, _lib.raw_stream(dev))


def _page_strides(k_pages, v_pages):
    """Strides of a layer's pages, checked."""
    if k_pages.ndim != 4 or v_pages.shape != k_pages.shape:
        raise ValueError("k_pages and v_pages must share a [pages, page_size, kv_heads, D] shape")
    if v_pages.dtype is not k_pages.dtype or v_pages.device != k_pages.device or not k_pages.is_cuda:
        raise ValueError("k_pages and v_pages must share type and CUDA device")
    ks, vs = k_pages.stride(), v_pages.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("the last dimension of k_pages and v_pages must be contiguous")
    return ks, vs


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
    not written, and ``status`` says so."""
    check_heads(k, "k")
    check_heads(v, "v", k)
    b, l, hkv, d = k.shape
    if v.shape[2] != hkv:
        raise ValueError("v must have k's shape")
    kps, vps = _page_strides(k_pages, v_pages)
    dev, dtype = k.device, DTYPES.get(k.dtype)
    if dtype is None or k_pages.dtype is not k.dtype or k_pages.device != dev:
        raise ValueError("k, v and the pages must share a type (BF16, FP16 or FP32) and a device")
    pages, page_size, ph, pd = k_pages.shape
    if ph != hkv or pd != d:
        raise ValueError(f"the pages hold heads of {(ph, pd)}, k has {(hkv, d)}")
    seqs = _ints(seqs, "seqs", 1, table.device)
    if seqs.shape[0] != b or table.device != dev:
        raise ValueError("seqs must name one sequence per batch row, on the tensors' device")
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {tuple(LAYOUTS)}, got {layout!r}")
    pairs, ip, pos = 0, 0, 0
    if inv_freq is not None:
        inv_freq, pairs = check_rotation(inv_freq, position_ids, b, l, d, layout, dev)
        ip = inv_freq.data_ptr()
        if position_ids is not None:
            if not position_ids.is_contiguous():
                position_ids = position_ids.contiguous()
            pos = position_ids.data_ptr()
    st = 0
    if start is not None:
        start = _ints(start, "start", 1, dev)
        if start.shape[0] != b:
            raise ValueError("start must hold one position per sequence")
        st = start.data_ptr()
    pt = _page_table(table, lengths, refcount, status, pages, page_size)
    k, v = inner_contiguous(k), inner_contiguous(v)
    qo, hq, qp, qop, qs = None, 0, 0, 0, (0, 0, 0)
    if q is not None:
        check_heads(q, "q", k)
        q = inner_contiguous(q)
        hq = q.shape[2]
        qo = new_heads(b, l, hq, d, k.dtype, dev)
        qp, qop, qs = q.data_ptr(), qo.data_ptr(), q.stride()
    ks, vs = k.stride(), v.stride()
    ra = _lib.ROTARY_ARGS.pack(qp, qop, k.data_ptr(), 0, pos, ip, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2],
                               b, l, hq, hkv, d, pairs, float(attention_factor), dtype, LAYOUTS[layout], 0)
    ap = _lib.APPEND_ARGS.pack(k_pages.data_ptr(), v_pages.data_ptr(), v.data_ptr(), seqs.data_ptr(), st,
                               kps[0], kps[1], kps[2], vps[0], vps[1], vps[2], vs[0], vs[1], vs[2],
                               0 if refcount is None else 1)
    _lib.call_packed("mrsa_paged_append", ra, pt, ap, _lib.raw_stream(dev))
    return qo


def paged_attention(q, k_pages, v_pages, table, lengths, seqs, *, causal: bool = False, key_valid=None,
                    scale: float | None = None, return_lse: bool = False, status=None):
    """Attention of ``q [B, L, Hq, D]`` (bf16 or fp16, D 64 or 128) over the
    cached tokens of the sequences ``seqs`` ``[B]`` in one layer's pages.

    The queries are a sequence's newest L tokens, whose keys and values the
    cache already holds: every query sees the whole sequence, as a block that
    is denoised does, or with ``causal`` the tokens up to its own position,
    ``length - L + i``.  ``key_valid`` (bool ``[B, max_pages * page_size]``)
    masks cached tokens; what masked tokens and unused slots hold does not
    matter.  Returns ``o [B, L, Hq, D]``, with ``return_lse`` also the
    natural-log LSE ``[B, L, Hq]`` in fp32; a query that sees no token gets
    zeros and -inf.  ``scale`` defaults to ``D ** -0.5``.  Forward only: it
    raises under autograd rather than return an output without a gradient."""
    check_heads(q, "q")
    ks, vs = _page_strides(k_pages, v_pages)
    b, l, hq, d = q.shape
    dev, qs = q.device, q.stride()
    pages, page_size, hkv, dk = k_pages.shape
    dtype = q.dtype
    if (dtype is not torch.bfloat16 and dtype is not torch.float16) or k_pages.dtype is not dtype or \
            k_pages.device != dev:
        raise ValueError("q and the pages must share a type (BF16 or FP16) and a device")
    if (d != 128 and d != 64) or dk != d or hkv < 1 or hq < hkv or hq % hkv:
        raise ValueError(f"heads must be of 64 or 128 dims, Hq a multiple of Hkv; got q {tuple(q.shape)}, "
                         f"pages {tuple(k_pages.shape)}")
    if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad):
        raise NotImplementedError("paged_attention is forward-only")
    seqs = _ints(seqs, "seqs", 1, table.device)
    if seqs.shape[0] != b or table.device != dev:
        raise ValueError("seqs must name one sequence per batch row, on the tensors' device")
    scale = d ** -0.5 if scale is None else float(scale)
    if not scale > 0:
        raise ValueError("scale must be positive")
    vp = 0
    if key_valid is not None:
        width = table.shape[1] * page_size
        if key_valid.dtype is not torch.bool or key_valid.shape != (b, width) or key_valid.device != dev:
            raise ValueError(f"key_valid must be bool {(b, width)} on the tensors' device")
        key_valid = _aligned(key_valid.contiguous())
        vp = key_valid.data_ptr()
    if qs[3] != 1 or (qs[0] | qs[1] | qs[2]) % 8 or q.data_ptr() % 16:
        q = _aligned(q.contiguous())
        qs = q.stride()
    pt = _page_table(table, lengths, None, status, pages, page_size)
    out = new_heads(b, l, hq, d, dtype, dev)
    lse, lp = None, 0
    if return_lse:
        lse = torch.empty_strided((b, l, hq), (l * hq, hq, 1), dtype=torch.float32, device=dev)
        lp = lse.data_ptr()
    args = _lib.PAGED_ATTENTION_ARGS.pack(
        q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), lp, vp, seqs.data_ptr(),
        qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], b, l, hq, hkv, d, scale, DTYPES[dtype], causal)
    size = _lib.load().mrsa_paged_attention_workspace(args)
    ws = torch.empty_strided((size,), (1,), dtype=torch.uint8, device=dev)
    _lib.call_packed("mrsa_paged_attention", args, pt, ws.data_ptr(), size, _lib.raw_stream(dev))
    return (out, lse) if return_lse else out


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
