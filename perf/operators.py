"""Rotary positions, the pages of a key-value cache, and the attention that reads them: cases to time and compare.

Each case runs one operator either in its plain form (elementary torch
operations in 32 bits, ``own = False``) or through the framework's public
entry points (``own = True``).  Both get the same inputs from ``prepare``.

Definitions.  *Rotary*: pair ``i`` of a head's first ``2 n`` dims turns by the
fp32 product ``position * inv_freq[i]`` (the angle the trained tables hold),
cosine and sine times a factor; the pair is dims ``(i, i + n)`` in the "half"
layout and ``(2i, 2i + 1)`` in the "interleaved" one; the dims past ``2 n``
pass through.  *Pages*: a pool ``[layers, 2, pages, page_size, kv_heads, D]``,
a table ``[sequences, max_pages]`` of page numbers (-1: none), lengths, and the
number of sequences that hold each page; a new page is always the lowest free
one, in the order of the call's sequences and then of their positions.
*Attention*: softmax over a sequence's cached tokens, natural-log LSE, zeros
and -inf for a row that sees nothing.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_framework = None


def _fw():
    """The framework's package (only where ``own`` is true)."""
    global _framework
    if _framework is None:
        import __graft_entry__

        _framework = __graft_entry__.load_package()
    return _framework


# ------------------------------------------------------------------ the cases
def listed():
    dream = {"hq": 28, "hkv": 4, "d": 128}
    return [
        # one denoising step's block of four sequences: the rotation by itself, where latency counts
        {"name": "rotary_block", "op": "rotary", "b": 4, "l": 32, **dream, "rot": 128, "layout": "half",
         "dtype": "bf16", "strided": True, "grad": False, "pos0": 4096},
        # a whole prompt's q and k, views of one fused projection's rows
        {"name": "rotary_prompt", "op": "rotary", "b": 1, "l": 16384, **dream, "rot": 128, "layout": "half",
         "dtype": "bf16", "strided": True, "grad": False, "pos0": 0},
        # a training step's rotation and its gradient: half of each head, neighbouring dims paired, odd length, fp32
        {"name": "rotary_train", "op": "rotary", "b": 2, "l": 4095, **dream, "rot": 64, "layout": "interleaved",
         "dtype": "fp32", "strided": False, "grad": True, "pos0": 0},
        # one new token of each of 64 sequences: q and k rotated, k and v into their pages
        {"name": "append_token", "op": "append", "b": 64, "l": 1, **dream, "rot": 128, "layout": "half",
         "dtype": "bf16", "page": 64, "lo": 1, "hi": 512, "heads_first": False},
        # a prompt's tokens into the cache of a layer, into pages of 16 with the heads outside
        {"name": "append_prompt", "op": "append", "b": 2, "l": 8191, **dream, "rot": 128, "layout": "half",
         "dtype": "bf16", "page": 16, "lo": 8191, "hi": 8300, "heads_first": True},
        # four candidate continuations of one prompt, its unfinished block copied in all layers, then one block more
        {"name": "fork_candidates", "op": "fork", "layers": 28, "sources": 1, "each": 4, "lo": 2021, "hi": 2021,
         "back": 32, "block": 32, "hkv": 4, "d": 128, "dtype": "bf16", "page": 64},
        # a long prompt thinned to half of its tokens for a continuation, in all layers
        {"name": "compact_prompt", "op": "compact", "layers": 28, "b": 2, "lo": 8190, "hi": 16384, "keep": 0.5,
         "hkv": 4, "d": 128, "dtype": "bf16", "page": 64},
        # one token over a short chat, where latency counts
        {"name": "attend_token_short", "op": "attend", "b": 1, "l": 1, **dream, "lo": 500, "hi": 500, "page": 64,
         "dtype": "bf16", "causal": False, "valid": 1.0, "heads_first": False, "strided": False},
        # one token of each of 64 sequences of all lengths
        {"name": "attend_token_batch", "op": "attend", "b": 64, "l": 1, **dream, "lo": 100, "hi": 16384, "page": 64,
         "dtype": "bf16", "causal": False, "valid": 1.0, "heads_first": False, "strided": False},
        # one token over one long document: the length has to be split
        {"name": "attend_token_long", "op": "attend", "b": 1, "l": 1, **dream, "lo": 131072, "hi": 131072, "page": 64,
         "dtype": "bf16", "causal": False, "valid": 1.0, "heads_first": False, "strided": False},
        # blocks of 32 tokens that see each other and all before them, some cached tokens masked
        {"name": "attend_block_batch", "op": "attend", "b": 8, "l": 32, **dream, "lo": 1000, "hi": 16384, "page": 64,
         "dtype": "fp16", "causal": False, "valid": 0.9, "heads_first": False, "strided": True},
        # one such block over a long document
        {"name": "attend_block_long", "op": "attend", "b": 1, "l": 32, **dream, "lo": 131072, "hi": 131072, "page": 64,
         "dtype": "bf16", "causal": False, "valid": 1.0, "heads_first": False, "strided": False},
    ]


def _between(rng, lo, hi):
    """A whole number spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    hq, hkv = rng.choice([(28, 4), (28, 4), (32, 8), (16, 16), (12, 1), (10, 2), (24, 8)])
    heads = {"hq": hq, "hkv": hkv}
    op = rng.choice(["rotary", "append", "fork", "compact", "attend", "attend", "attend"])
    if op == "rotary":
        b, d = rng.choice([1, 1, 2, 3]), rng.choice([64, 128, 128, 256])
        return {"op": op, "b": b, "l": _between(rng, 1, 3000) if b > 1 else _between(rng, 1, 12000), **heads, "d": d,
                "rot": rng.choice([d, d, d // 2, d // 4]), "layout": rng.choice(["half", "interleaved"]),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "strided": rng.random() < 0.5,
                "grad": rng.random() < 0.4, "pos0": rng.choice([0, 1000, 130000])}
    if op == "append":
        d, b = rng.choice([64, 128]), _between(rng, 1, 64)
        n = _between(rng, 1, max(1, 6000 // b))
        lo = n + rng.randrange(40)
        return {"op": op, "b": b, "l": n, **heads, "d": d, "rot": rng.choice([d, d, d // 2]),
                "layout": rng.choice(["half", "interleaved"]), "dtype": rng.choice(["bf16", "fp16"]),
                "page": rng.choice([16, 32, 64, 128]), "lo": lo, "hi": lo + _between(rng, 1, 300),
                "heads_first": rng.random() < 0.5}
    if op == "fork":
        lo = _between(rng, 1, 4000)
        return {"op": op, "layers": rng.choice([1, 4, 28]), "sources": rng.choice([1, 2, 3]),
                "each": _between(rng, 1, 8), "lo": lo, "hi": lo + rng.randrange(300), "back": rng.choice([0, 1, 32, 100]),
                "block": rng.choice([1, 32, 65]), "hkv": hkv if hkv < 16 else 8, "d": rng.choice([64, 128]),
                "dtype": rng.choice(["bf16", "fp16"]), "page": rng.choice([16, 32, 64, 128])}
    if op == "compact":
        lo = _between(rng, 1, 3000)
        return {"op": op, "layers": rng.choice([1, 4, 28]), "b": rng.choice([1, 2, 5]), "lo": lo,
                "hi": lo + rng.randrange(1500), "keep": rng.choice([0.0, 0.1, 0.5, 0.95, 1.0]),
                "hkv": hkv if hkv < 16 else 8, "d": rng.choice([64, 128]), "dtype": rng.choice(["bf16", "fp16"]),
                "page": rng.choice([16, 32, 64, 128])}
    d, l = rng.choice([64, 128, 128]), rng.choice([1, 1, 1, 2, 3, 5, 16, 32, 33, 100])
    b = _between(rng, 1, 48)
    hi = _between(rng, 1, 100000 // b * 4 // max(4, hkv) // (3 if l > 33 else 1))
    return {"op": op, "b": b, "l": l, **heads, "lo": rng.choice([0, 1, hi // 2, hi]), "hi": hi, "d": d,
            "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["bf16", "fp16"]),
            "causal": l > 1 and rng.random() < 0.4, "valid": rng.choice([1.0, 1.0, 0.9, 0.3]),
            "heads_first": rng.random() < 0.4, "strided": rng.random() < 0.5}


def _lengths(c, n):
    """``n`` lengths spread over [lo, hi], the first the shortest and the second the longest."""
    lo, hi = c["lo"], c["hi"]
    got = [lo + int((hi - lo + 1) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]
    return got if n < 2 else [lo, hi] + got[2:]


def _lens(c):
    if c["op"] == "fork":
        return _lengths(c, c["sources"])
    return [max(c["lo"], c["hi"])] if c["b"] == 1 and c["op"] != "append" else _lengths(c, c["b"])


# ------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)


def _inv_freq(n):
    """Inverse frequencies of a context scaled eightfold (base 1e6), fast ones kept, slow ones divided, and the factor."""
    i = torch.arange(n, dtype=torch.float32)
    f = 1.0e6 ** (-i / n)
    keep = (1 - (i / n - 0.15) / 0.25).clamp(0, 1)
    return (f * keep + f / 8 * (1 - keep)).cuda(), 0.1 * math.log(8.0) + 1.0


def _heads(g, c, dtype, strided, *counts):
    """Tensors [b, l, n, d] for each n of counts: views of one fused projection's rows, or tensors of their own."""
    b, l, d = c["b"], c["l"], c["d"]
    if strided:
        x = _randn(g, b, l, sum(counts), d, dtype=dtype)
        return torch.split(x, list(counts), dim=2)
    return [_randn(g, b, l, n, d, dtype=dtype) for n in counts]


def _table(g, lens, page, width, pages):
    """The table [n, width] of sequences whose pages are scattered over the pool."""
    n = len(lens)
    held = torch.tensor([-(-x // page) for x in lens], device="cuda")
    j = torch.arange(width, device="cuda")
    has = j < held[:, None]
    order = torch.randperm(pages, device="cuda", generator=g)
    rank = (has.flatten().cumsum(0) - 1).clamp_min(0).view(n, width)
    return torch.where(has, order[rank], torch.full_like(rank, -1)).to(torch.int32)


def _counts(table, pages):
    """How many sequences hold each page."""
    got = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    flat = torch.where(table < 0, torch.full_like(table, pages), table).flatten().long()
    return got.index_add_(0, flat, torch.ones_like(flat, dtype=torch.int32))[:pages].contiguous()


def prepare(case, seed):
    c = case
    g = _generator(seed)
    dtype = _DTYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "rotary":
        q, k = _heads(g, c, dtype, c["strided"], c["hq"], c["hkv"])
        pos = c["pos0"] + torch.arange(c["l"], device="cuda")
        inv, factor = _inv_freq(c["rot"] // 2)
        # positions as a cache with one summary slot a chunk numbers them: the slots share their neighbour's
        s |= {"q": q, "k": k, "pos": (pos - pos // 64).expand(c["b"], c["l"]).contiguous(), "inv": inv, "factor": factor}
        if c["grad"]:
            s["gq"], s["gk"] = _heads(g, c, dtype, False, c["hq"], c["hkv"])
            s["q"], s["k"] = q.detach().requires_grad_(), k.detach().requires_grad_()
        return s
    lens, page = _lens(c), c["page"]
    if c["op"] in ("fork", "compact"):
        extra = c["sources"] * c["each"] if c["op"] == "fork" else c["b"]
        n = len(lens)
        width = max(-(-(x + c.get("block", 0)) // page) for x in lens) + 1
        held = [-(-x // page) for x in lens]
        pages = sum(held) + 3
        if c["op"] == "fork":
            pages += c["each"] * sum(h + 2 + c["block"] // page - max(0, x - c["back"]) // page for h, x in zip(held, lens))
        else:
            pages += sum(held) + 2 * n
        pool = _randn(g, c["layers"], 2, pages, page, c["hkv"], c["d"], dtype=dtype)
        table = torch.full((n + extra, width), -1, dtype=torch.int32, device="cuda")
        table[:n] = _table(g, lens, page, width, pages)
        lengths = torch.zeros(n + extra, dtype=torch.int32, device="cuda")
        lengths[:n] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s |= {"pool": pool, "table": table, "lengths": lengths, "refcount": _counts(table, pages)}
        src = torch.arange(n, device="cuda", dtype=torch.int32)
        s["dst"] = torch.arange(n, n + extra, device="cuda", dtype=torch.int32)
        s["src"] = src.repeat_interleave(c["each"]) if c["op"] == "fork" else src
        if c["op"] == "fork":
            s["share"] = (lengths[s["src"].long()] - c["back"]).clamp_min(0)
            s["copies"] = c["each"] * sum(h - max(0, x - c["back"]) // page for h, x in zip(held, lens))
            s["grown"] = sum(-(-(x + c["block"]) // page) - h for h, x in zip(held, lens)) * c["each"]
        else:
            # whole chunks are kept or thinned, as an importance score over chunks gives them
            near = torch.rand(n, -(-width * page // 64), device="cuda", generator=g).repeat_interleave(64, 1)
            each = torch.rand(n, width * page, device="cuda", generator=g)
            x = c["keep"]
            below = math.sqrt(2 * x) if x < 0.5 else 2 - math.sqrt(2 * (1 - x))  # so that a share x of the sums is
            s["keep"] = near[:, :width * page] + each < below
        return s
    width = max(1, max(-(-x // page) for x in lens))
    pages = sum(-(-x // page) for x in lens) + 2
    s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["table"] = _table(g, lens, page, width, pages)
    shape = (2, pages, c["hkv"], page, c["d"]) if c["heads_first"] else (2, pages, page, c["hkv"], c["d"])
    pool = _randn(g, *shape, dtype=dtype)
    if c["heads_first"]:
        pool = pool.transpose(2, 3)
    s["k_pages"], s["v_pages"] = pool[0], pool[1]
    perm = torch.randperm(c["b"], device="cuda", generator=g)
    s["seqs"] = perm.to(torch.int32)
    if c["op"] == "append":
        s["q"], s["k"], s["v"] = _heads(g, c, dtype, True, c["hq"], c["hkv"], c["hkv"])
        at = s["lengths"][perm].long()[:, None] - c["l"] + torch.arange(c["l"], device="cuda")
        s["pos"] = (at - at // 64).contiguous()
        s["inv"], s["factor"] = _inv_freq(c["rot"] // 2)
        s["refcount"] = _counts(s["table"], pages)
        return s
    q, = _heads(g, c, dtype, False, c["hq"] + (2 * c["hkv"] if c["strided"] else 0))
    s["q"] = (q * 1.5)[:, :, :c["hq"]]  # logits of a spread that makes some tokens stand out
    s["valid"] = None
    if c["valid"] < 1.0:
        s["valid"] = torch.rand(c["b"], width * page, device="cuda", generator=g) < c["valid"]
    return s


# ------------------------------------------------------------------ plain forms
def _rotate(x, pos, inv, factor, layout):
    """x [b, l, h, d] in 32 bits, its first 2 * len(inv) dims rotated."""
    angle = (pos.to(torch.float32)[..., None] * inv)[:, :, None]
    cos, sin = angle.cos() * factor, angle.sin() * factor
    n = inv.shape[0]
    x = x.to(torch.float32)
    if layout == "half":
        a, b = x[..., :n], x[..., n:2 * n]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, x[..., 2 * n:]), -1)


def _plain_rotary(s):
    c = s["case"]
    dtype = _DTYPES[c["dtype"]]
    yq = _rotate(s["q"], s["pos"], s["inv"], s["factor"], c["layout"]).to(dtype)
    yk = _rotate(s["k"], s["pos"], s["inv"], s["factor"], c["layout"]).to(dtype)
    if not c["grad"]:
        return yq, yk
    return (yq, yk) + torch.autograd.grad((yq, yk), (s["q"], s["k"]), (s["gq"], s["gk"]))


def _plain_append(s):
    c = s["case"]
    dtype, page = _DTYPES[c["dtype"]], c["page"]
    q = _rotate(s["q"], s["pos"], s["inv"], s["factor"], c["layout"]).to(dtype)
    k = _rotate(s["k"], s["pos"], s["inv"], s["factor"], c["layout"]).to(dtype)
    seqs = s["seqs"].long()
    at = s["lengths"][seqs].long()[:, None] - c["l"] + torch.arange(c["l"], device=q.device)
    where = s["table"][seqs[:, None], at // page].long()
    s["k_pages"][where, at % page] = k
    s["v_pages"][where, at % page] = s["v"]
    return q, s["k_pages"], s["v_pages"]


def _release(table, lengths, refcount, seqs):
    rows = table[seqs].flatten().long()
    refcount.index_add_(0, rows.clamp_min(0), -(rows >= 0).to(torch.int32))
    table[seqs] = -1
    lengths[seqs] = 0


def _new_pages(refcount, wanted):
    """The lowest free pages, one for each place of the mask that wants one, in order; -1 elsewhere."""
    free = torch.argsort((refcount != 0).to(torch.int32), stable=True)
    rank = (wanted.flatten().cumsum(0) - 1).clamp_min(0).view(wanted.shape)
    got = torch.where(wanted, free[rank], torch.full_like(rank, -1))
    refcount.index_add_(0, got.flatten().clamp_min(0), wanted.flatten().to(torch.int32))
    return got


def _plain_share(s, share):
    """The sources' pages for dst: those below share tokens are held in common, the others are copied."""
    table, lengths, refcount, pool, page = s["table"], s["lengths"], s["refcount"], s["pool"], s["case"]["page"]
    src, dst = s["src"].long(), s["dst"].long()
    _release(table, lengths, refcount, dst)
    n = lengths[src].long()
    j = torch.arange(table.shape[1], device=table.device)
    rows = table[src].long()
    common = j < (torch.minimum(share.long(), n) // page)[:, None]
    apart = (j < ((n + page - 1) // page)[:, None]) & ~common
    refcount.index_add_(0, rows.flatten().clamp_min(0), common.flatten().to(torch.int32))
    new = _new_pages(refcount, apart)
    table[dst] = torch.where(common, rows, new).to(torch.int32)
    lengths[dst] = n.to(torch.int32)
    return rows, new, apart


def _plain_fork(s):
    c = s["case"]
    table, lengths, refcount, pool, page = s["table"], s["lengths"], s["refcount"], s["pool"], c["page"]
    rows, new, apart = _plain_share(s, s["share"])
    pick = torch.argsort((~apart).flatten().to(torch.int32), stable=True)[:s["copies"]]
    pool[:, :, new.flatten()[pick]] = pool[:, :, rows.flatten()[pick]]
    dst = s["dst"].long()
    n = lengths[dst].long()
    j = torch.arange(table.shape[1], device=table.device)
    grown = (j >= ((n + page - 1) // page)[:, None]) & (j < ((n + c["block"] + page - 1) // page)[:, None])
    more = _new_pages(refcount, grown)
    table[dst] = torch.where(grown, more.to(torch.int32), table[dst])
    lengths[dst] = (n + c["block"]).to(torch.int32)
    return pool, table, lengths, refcount


def _plain_compact(s):
    table, lengths, refcount, pool, page = s["table"], s["lengths"], s["refcount"], s["pool"], s["case"]["page"]
    rows, new, apart = _plain_share(s, s["lengths"][s["src"].long()])
    pick = apart.flatten().nonzero().flatten()
    pool[:, :, new.flatten()[pick]] = pool[:, :, rows.flatten()[pick]]
    dst = s["dst"].long()
    n, w = lengths[dst].long(), table.shape[1]
    at = torch.arange(w * page, device=table.device)
    inside = at < n[:, None]
    keep = s["keep"] & inside
    left = keep.sum(1)
    # pages before a sequence's first dropped token stay; the kept tokens after them go to new pages
    first = torch.where(inside & ~keep, at, w * page).amin(1) // page
    stay = torch.minimum(first, (n + page - 1) // page)
    stay = torch.where(left == n, (n + page - 1) // page, stay)
    j = torch.arange(w, device=table.device)
    old = table[dst].long()
    wanted = (j >= stay[:, None]) & (j < ((left + page - 1) // page)[:, None])
    dropped = (j >= stay[:, None]) & (old >= 0)
    fresh = _new_pages(refcount, wanted)
    move = keep & (at >= (stay * page)[:, None])
    i, source = move.nonzero(as_tuple=True)
    target = (keep.to(torch.int32).cumsum(1) - 1)[i, source].long()
    pool[:, :, fresh[i, target // page], target % page] = pool[:, :, old[i, source // page], source % page]
    refcount.index_add_(0, old.flatten().clamp_min(0), -dropped.flatten().to(torch.int32))
    table[dst] = torch.where(j < stay[:, None], old, fresh).to(torch.int32)
    lengths[dst] = left.to(torch.int32)
    return pool, table, lengths, refcount


def _plain_attend(s):
    c = s["case"]
    q, page = s["q"], c["page"]
    b, l, hq, d = q.shape
    hkv = c["hkv"]
    seqs = s["seqs"].long()
    n = s["lengths"][seqs].long()
    rows = s["table"][seqs].long().clamp_min(0)
    at = torch.arange(rows.shape[1] * page, device=q.device)
    cached = at < n[:, None]
    if s["valid"] is not None:
        cached = cached & s["valid"]

    def tokens(pages):  # [b, hkv, tokens, d], zeros where there is no token
        x = pages[rows].flatten(1, 2).transpose(1, 2).to(torch.float32)
        return torch.where(cached[:, None, :, None], x, torch.zeros((), device=x.device))

    x = q.to(torch.float32).view(b, l, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)
    scores = (x @ tokens(s["k_pages"]).transpose(-1, -2)) * d ** -0.5
    seen = cached[:, None, None]
    if c["causal"]:
        own_at = n[:, None] - l + torch.arange(l, device=q.device)
        seen = seen & (at <= own_at[:, :, None])[:, None].repeat_interleave(hq // hkv, 2)
    scores = torch.where(seen, scores, torch.full((), -math.inf, device=q.device))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = (p @ tokens(s["v_pages"])) / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + torch.log(total))[..., 0]
    o = o.view(b, hkv, l, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, l, hq, d)
    lse = lse.view(b, hkv, l, hq // hkv).permute(0, 2, 1, 3).reshape(b, l, hq)
    return o.to(q.dtype), lse


_PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "fork": _plain_fork, "compact": _plain_compact,
          "attend": _plain_attend}


# ------------------------------------------------------------------ the framework's calls
def _own_rotary(s):
    c = s["case"]
    yq, yk = _fw().rotary_embedding(s["q"], s["k"], s["pos"], s["inv"], s["factor"], layout=c["layout"])
    if not c["grad"]:
        return yq, yk
    return (yq, yk) + torch.autograd.grad((yq, yk), (s["q"], s["k"]), (s["gq"], s["gk"]))


def _own_append(s):
    q = _fw().paged_append(s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["seqs"], s["k"], s["v"], q=s["q"],
                           position_ids=s["pos"], inv_freq=s["inv"], attention_factor=s["factor"],
                           layout=s["case"]["layout"], refcount=s["refcount"])
    return q, s["k_pages"], s["v_pages"]


def _own_fork(s):
    fw = _fw()
    state = s["table"], s["lengths"], s["refcount"]
    fw.page_fork(s["pool"], *state, s["src"], s["dst"], s["share"])
    fw.page_extend(*state, s["dst"], s["case"]["block"], page_size=s["case"]["page"])
    return (s["pool"],) + state


def _own_compact(s):
    fw = _fw()
    state = s["table"], s["lengths"], s["refcount"]
    fw.page_free(*state, s["dst"])
    fw.page_fork(s["pool"], *state, s["src"], s["dst"])
    fw.page_compact(s["pool"], *state, s["dst"], s["keep"])
    return (s["pool"],) + state


def _own_attend(s):
    return _fw().paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["seqs"],
                                 causal=s["case"]["causal"], key_valid=s["valid"], return_lse=True)


_OWN = {"rotary": _own_rotary, "append": _own_append, "fork": _own_fork, "compact": _own_compact,
        "attend": _own_attend}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    e = _BYTES[c["dtype"]]
    if c["op"] == "rotary":
        n = c["b"] * c["l"] * (c["hq"] + c["hkv"])
        times = 2 if c["grad"] else 1
        return {"bytes": times * (2 * n * c["d"] * e + 8 * c["b"] * c["l"]), "flops": times * 3 * n * c["rot"]}
    lens, page = _lens(c), c["page"]
    if c["op"] == "append":
        t = c["b"] * c["l"]
        return {"bytes": t * ((2 * c["hq"] + 4 * c["hkv"]) * c["d"] * e + 8),
                "flops": 3 * t * (c["hq"] + c["hkv"]) * c["rot"]}
    token = 2 * c.get("layers", 1) * c["hkv"] * c["d"] * e if c["op"] != "attend" else 2 * c["hkv"] * c["d"] * e
    held = [-(-x // page) for x in lens]
    if c["op"] == "fork":
        copied = c["each"] * sum(h - max(0, x - c["back"]) // page for h, x in zip(held, lens))
        return {"bytes": 2 * copied * page * token + 8 * c["each"] * sum(held), "flops": 0}
    if c["op"] == "compact":
        part = sum(x % page for x in lens)
        kept = (c["keep"] if c["keep"] < 1.0 else 0.0) * sum(lens)  # about: nothing moves where all is kept
        return {"bytes": 2 * (part + kept) * token + sum(lens) + 8 * sum(held), "flops": 0}
    rows = c["b"] * c["l"] * c["hq"]
    seen = sum(lens) * c["l"] - (sum(min(x, c["l"]) * (c["l"] - 1) // 2 for x in lens) if c["causal"] else 0)
    return {"bytes": sum(lens) * (token + (1 if c["valid"] < 1.0 else 0)) + rows * (2 * c["d"] * e + 4),
            "flops": max(1, 4 * seen * c["hq"] * c["d"])}


# ------------------------------------------------------------------ the definition in 64 bits
def _turn64(x, pos, inv, factor, layout, sign=1.0):
    """x [b, l, h, d]: each pair as a complex number times factor * exp(i angle)."""
    angle = (pos.to(torch.float32)[..., None] * inv).double()[:, :, None, :]  # the angle is the fp32 product
    w = torch.polar(torch.full_like(angle, factor), sign * angle)
    n = inv.shape[0]
    out = x.detach().double().clone()
    r = slice(0, n) if layout == "half" else slice(0, 2 * n, 2)
    i = slice(n, 2 * n) if layout == "half" else slice(1, 2 * n, 2)
    z = torch.complex(out[..., r], out[..., i]) * w
    out[..., r], out[..., i] = z.real, z.imag
    return out


def exact(case, seed):
    c = case
    if c["op"] in ("fork", "compact"):
        return None  # copies and whole numbers
    s = prepare(c, seed)
    if c["op"] == "rotary":
        rot = (s["pos"], s["inv"], s["factor"], c["layout"])
        got = [_turn64(s["q"], *rot), _turn64(s["k"], *rot)]
        if c["grad"]:
            got += [_turn64(s["gq"], *rot, sign=-1.0), _turn64(s["gk"], *rot, sign=-1.0)]
        return tuple(got)
    page = c["page"]
    lens, seqs, table = s["lengths"].tolist(), s["seqs"].tolist(), s["table"].tolist()
    if c["op"] == "append":
        rot = (s["pos"], s["inv"], s["factor"], c["layout"])
        k, kp, vp = _turn64(s["k"], *rot), s["k_pages"].double(), s["v_pages"].double()
        for i, row in enumerate(seqs):
            slots = [table[row][a // page] * page + a % page for a in range(lens[row] - c["l"], lens[row])]
            slots = torch.tensor(slots, device="cuda")
            kp[slots // page, slots % page] = k[i]
            vp[slots // page, slots % page] = s["v"][i].double()
        return _turn64(s["q"], *rot), kp, vp
    o = torch.zeros(c["b"], c["l"], c["hq"], c["d"], dtype=torch.float64, device="cuda")
    lse = torch.full((c["b"], c["l"], c["hq"]), -math.inf, dtype=torch.float64, device="cuda")
    group = c["hq"] // c["hkv"]
    for i, row in enumerate(seqs):
        n = lens[row]
        if n == 0:
            continue
        held = torch.tensor(table[row][:-(-n // page)], device="cuda")
        at = torch.arange(n, device="cuda")
        use = torch.ones(n, dtype=torch.bool, device="cuda") if s["valid"] is None else s["valid"][i, :n]
        for h in range(c["hkv"]):
            k = s["k_pages"][held, :, h].flatten(0, 1)[:n][use].double()
            v = s["v_pages"][held, :, h].flatten(0, 1)[:n][use].double()
            x = s["q"][i, :, h * group:(h + 1) * group].double()  # [l, group, d]
            logits = torch.einsum("lgd,td->lgt", x, k) / math.sqrt(c["d"])
            if c["causal"]:
                late = at[use][None, :] > (n - c["l"] + torch.arange(c["l"], device="cuda"))[:, None]
                logits = logits.masked_fill(late[:, None, :], -math.inf)
            if k.shape[0] == 0:
                continue
            o[i, :, h * group:(h + 1) * group] = torch.einsum("lgt,td->lgd", logits.softmax(-1), v).nan_to_num(0.0)
            lse[i, :, h * group:(h + 1) * group] = torch.logsumexp(logits, -1)
    return o, lse
