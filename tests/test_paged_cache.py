"""Pages of a key-value cache (``paged_cache.py``): the table's bookkeeping
against a plain model of it on the host, the pages' contents against their
definition, what is refused and reported, and the rotated append against the
formula in 64 bits (bounds as in ``test_rotary.py``).  Whole numbers and
copied bytes are equal, bit for bit."""

import random

import pytest
import torch

from test_rotary import check as check_turned


class Model:
    """The definition of the page operators on Python lists; `tokens[s]` are
    the tokens that a sequence holds."""

    def __init__(self, sequences, max_pages, pages, page_size):
        self.rows = [[] for _ in range(sequences)]
        self.tokens = [[] for _ in range(sequences)]
        self.count = [0] * pages
        self.width, self.ps = max_pages, page_size

    def lowest(self, n):
        free = [p for p, c in enumerate(self.count) if c == 0]
        return free[:n] if len(free) >= n else None

    def free(self, seqs):
        for s in seqs:
            for p in self.rows[s]:
                self.count[p] -= 1
            self.rows[s], self.tokens[s] = [], []

    def take(self, pages):
        for p in pages:
            self.count[p] += 1

    def extend(self, seqs, more):
        want = [-(-(len(self.tokens[s]) + m) // self.ps) - len(self.rows[s]) for s, m in zip(seqs, more)]
        if any(len(self.rows[s]) + w > self.width for s, w in zip(seqs, want)):
            return 4
        new = self.lowest(sum(want))
        if new is None:
            return 2
        self.take(new)
        for s, m, w in zip(seqs, more, want):
            self.rows[s] += new[:w]
            new = new[w:]
            self.tokens[s] += [None] * m
        return 0

    def fork(self, src, dst, share):
        self.free(dst)
        common = [min(h, len(self.tokens[s])) // self.ps for s, h in zip(src, share)]
        new = self.lowest(sum(len(self.rows[s]) - c for s, c in zip(src, common)))
        if new is None:
            return 2
        for s, d, c in zip(src, dst, common):
            n = len(self.rows[s]) - c
            self.rows[d] = self.rows[s][:c] + new[:n]
            self.take(self.rows[d])
            new = new[n:]
            self.tokens[d] = list(self.tokens[s])
        return 0

    def compact(self, seqs, keep):
        plan = []
        for s, k in zip(seqs, keep):
            n = len(self.tokens[s])
            drop = [i for i in range(n) if not k[i]]
            stay = drop[0] // self.ps if drop else len(self.rows[s])
            left = [t for t, m in zip(self.tokens[s], k) if m]
            plan.append((s, stay, left, -(-len(left) // self.ps) - stay))
        new = self.lowest(sum(p[3] for p in plan))
        if new is None:
            return 2
        self.take(new)
        for s, stay, left, n in plan:
            for p in self.rows[s][stay:]:
                self.count[p] -= 1
            self.rows[s] = self.rows[s][:stay] + new[:n]
            new = new[n:]
            self.tokens[s] = left
        return 0

    def same(self, cache):
        table = [r + [-1] * (self.width - len(r)) for r in self.rows]
        assert cache.table.tolist() == table
        assert cache.lengths.tolist() == [len(t) for t in self.tokens]
        assert cache.refcount.tolist() == self.count

    def same_tokens(self, cache):
        """Every plane's slot of every known token holds that token's number."""
        first = cache.pool[..., 0, 0].float()       # [layers, 2, pages, page_size]
        for row, toks in zip(self.rows, self.tokens):
            at = [(row[i // self.ps], i % self.ps, t) for i, t in enumerate(toks) if t is not None]
            if at:
                p, s, t = (torch.tensor(x, device=first.device) for x in zip(*at))
                assert (first[:, :, p, s] == t).all()


def numbered(mrsa, model, cache, seqs, rng):
    """Gives the last tokens of seqs (those without one) a number of their own, through append, in every layer."""
    dev = cache.table.device
    layers, _, _, ps, h, d = cache.pool.shape
    for s in seqs:
        toks = model.tokens[s]
        new = [i for i, t in enumerate(toks) if t is None]
        if not new:
            continue
        for i in new:
            toks[i] = rng.randrange(1, 250)         # whole numbers that bf16 holds
        x = torch.tensor([toks[i] for i in new], device=dev, dtype=cache.pool.dtype)
        x = x.view(1, -1, 1, 1).expand(1, len(new), h, d)
        for layer in range(layers):
            cache.append(layer, cache.seqs(s), x, x, start=torch.tensor([new[0]], dtype=torch.int32, device=dev))


@pytest.mark.gpu
@pytest.mark.parametrize("page_size,layers,heads,dtype,outside", [
    (16, 2, 3, torch.bfloat16, "tokens"), (64, 1, 1, torch.float16, "tokens"), (32, 3, 2, torch.bfloat16, "heads")])
def test_random_calls_match_the_model(mrsa, cuda_device, page_size, layers, heads, dtype, outside):
    rng = random.Random(page_size)
    sequences, width, pages = 7, 9, 30
    cache = mrsa.PagedKVCache(layers, pages, heads, 64, sequences=sequences, max_len=width * page_size,
                              page_size=page_size, dtype=dtype, device=cuda_device)
    if outside == "heads":
        cache.pool = torch.empty(layers, 2, pages, heads, page_size, 64, dtype=dtype, device=cuda_device).transpose(3, 4)
    cache.pool.fill_(float("nan"))
    model = Model(sequences, width, pages, page_size)
    dev = cuda_device
    reports = 0
    for step in range(60):
        kind = rng.choice(["extend", "extend", "fork", "compact", "free"])
        n = rng.randint(1, 3)
        if kind == "fork":
            src = [rng.randrange(sequences) for _ in range(n)]
            dst = rng.sample([s for s in range(sequences) if s not in src], n)
            share = [rng.randrange(0, width * page_size) for _ in src]
            given = None if step % 3 == 0 else torch.tensor(share, dtype=torch.int32, device=dev)
            if given is None:
                share = [len(model.tokens[s]) for s in src]
            cache.fork(cache.seqs(*src), cache.seqs(*dst), given)
            want = model.fork(src, dst, share)
        else:
            seqs = rng.sample(range(sequences), n)
            if kind == "extend":
                more = [rng.randrange(0, 3 * page_size) for _ in seqs]
                if step % 2:
                    more = [more[0]] * n
                cache.extend(cache.seqs(*seqs), more[0] if step % 2 else torch.tensor(more, dtype=torch.int32, device=dev))
                want = model.extend(seqs, more)
            elif kind == "compact":
                p = rng.choice([0.0, 0.5, 0.97, 1.0])
                keep = [[rng.random() < p for _ in range(width * page_size)] for _ in seqs]
                cache.compact(cache.seqs(*seqs), torch.tensor(keep, device=dev))
                want = model.compact(seqs, keep)
            else:
                cache.free(cache.seqs(*seqs))
                want = model.free(seqs) or 0
        assert cache.status.item() == want, (step, kind)
        cache.status.zero_()
        reports += want != 0
        model.same(cache)
        numbered(mrsa, model, cache, range(sequences) if kind == "extend" and not want else [], rng)
        assert cache.status.item() in (0,), (step, kind)
        model.same_tokens(cache)
    assert reports < 40           # the calls that did not fit said so, and most did fit


@pytest.mark.gpu
def test_many_sequences_and_a_large_pool(mrsa, cuda_device):
    """More sequences than groups of threads, a free list across all CTAs, rows longer than a CTA has threads."""
    rng = random.Random(5)
    ps, sequences, width, pages = 16, 300, 1500, 40000
    cache = mrsa.PagedKVCache(1, pages, 1, 8, sequences=sequences, max_len=width * ps, page_size=ps, device=cuda_device)
    model = Model(sequences, width, pages, ps)
    some = rng.sample(range(sequences), 150)
    lens = [rng.choice([0, 1, 15, 16, 17, 700, 3000]) for _ in some]
    lens[3] = width * ps - 5
    cache.extend(cache.seqs(*some), torch.tensor(lens, dtype=torch.int32, device=cuda_device))
    assert model.extend(some, lens) == 0
    model.same(cache)
    numbered(mrsa, model, cache, some[:20], rng)
    out = some[::2]
    cache.free(cache.seqs(*out))
    model.free(out)
    rest = [s for s in range(sequences) if s not in some]
    src = [some[2 * i + 1] for i in range(70)]
    share = [rng.randrange(3200) for _ in src]
    cache.fork(cache.seqs(*src), cache.seqs(*rest[:70]), torch.tensor(share, dtype=torch.int32, device=cuda_device))
    assert model.fork(src, rest[:70], share) == 0
    model.same(cache)
    who = [some[3]] + rest[:69]
    keep = [[rng.random() < 0.6 for _ in range(width * ps)] for _ in who]
    cache.compact(cache.seqs(*who), torch.tensor(keep, device=cuda_device))
    assert model.compact(who, keep) == 0
    cache.check()
    model.same(cache)
    model.same_tokens(cache)


@pytest.mark.gpu
def test_what_cannot_be_done_is_reported(mrsa, cuda_device):
    dev = cuda_device
    cache = mrsa.PagedKVCache(1, 6, 1, 64, sequences=4, max_len=64, page_size=16, device=dev)
    cache.extend(cache.seqs(0, 1), 40)                       # three pages each
    before = [cache.table.tolist(), cache.lengths.tolist(), cache.refcount.tolist()]

    def unchanged(exc, match):
        with pytest.raises(exc, match=match):
            cache.check()
        assert [cache.table.tolist(), cache.lengths.tolist(), cache.refcount.tolist()] == before
        cache.check()                                        # the word was cleared

    cache.extend(cache.seqs(2), 1)
    unchanged(RuntimeError, "free pages")
    cache.extend(cache.seqs(0), 25)
    unchanged(ValueError, "outgrow")
    cache.extend(cache.seqs(2, 2), 1)
    unchanged(ValueError, "twice")
    cache.free(cache.seqs(0, 4))
    unchanged(ValueError, "out of range")
    cache.free(cache.seqs(-1))
    unchanged(ValueError, "out of range")
    cache.fork(cache.seqs(0), cache.seqs(0))
    unchanged(ValueError, "twice")
    cache.fork(cache.seqs(0, 1), cache.seqs(2, 1))
    unchanged(ValueError, "twice")
    keep = torch.zeros(1, 64, dtype=torch.bool, device=dev)
    keep[0, 1:] = True
    cache.compact(cache.seqs(0), keep)                       # needs three new pages
    unchanged(RuntimeError, "free pages")
    # a fork that does not fit leaves its targets empty
    cache.fork(cache.seqs(0), cache.seqs(2))
    with pytest.raises(RuntimeError, match="free pages"):
        cache.check()
    assert cache.lengths.tolist() == [40, 40, 0, 0] and cache.table[2].tolist() == [-1] * 4
    # whole pages in common need no new one; a write to them is refused, elsewhere it is not
    cache.free(cache.seqs(1))
    cache.fork(cache.seqs(0), cache.seqs(3))
    x = torch.ones(1, 1, 1, 64, dtype=torch.bfloat16, device=dev)
    cache.pool.zero_()
    cache.append(0, cache.seqs(3), x, x, start=torch.tensor([31], dtype=torch.int32, device=dev))
    with pytest.raises(ValueError, match="several sequences"):
        cache.check()
    assert not cache.pool.any()
    cache.append(0, cache.seqs(3), x, x)
    cache.check()
    assert cache.pool[0, :, cache.table[3, 2], 7].eq(1).all() and cache.pool.sum() == 128
    for s, start in ((3, 40), (3, -1), (2, 0), (9, 0)):
        cache.append(0, cache.seqs(s), x, x, start=torch.tensor([start], dtype=torch.int32, device=dev))
        with pytest.raises(ValueError):
            cache.check()
    assert cache.pool.sum() == 128


@pytest.mark.gpu
def test_copy_pages(mrsa, cuda_device):
    dev = cuda_device
    for pool in (torch.randn(3, 2, 9, 16, 5, 24, device=dev), torch.randn(2, 2, 9, 5, 16, 8, device=dev).bfloat16().transpose(3, 4)):
        want = pool.clone()
        want[:, :, [0, 7, 3]] = pool[:, :, [4, 4, 8]]
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        t = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        mrsa.page_copy(pool, t(4, 4, 8), t(0, 7, 3), status=status)
        assert torch.equal(pool, want) and status.item() == 0
        mrsa.page_copy(pool, t(9, 4, -1), t(0, 9, 3), status=status)
        assert torch.equal(pool, want) and status.item() == 8
        mrsa.page_copy(pool, t(), t())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,l,hq,hk,d,n,page,heads_first,layout", [
    (3, 1, 28, 4, 128, 64, 64, False, "half"), (2, 37, 6, 2, 64, 16, 16, True, "interleaved"),
    (1, 130, 2, 2, 80, 10, 32, False, "half"), (4, 3, 0, 1, 24, 0, 16, True, "half")])
def test_append_rotates_and_writes(mrsa, cuda_device, dtype, b, l, hq, hk, d, n, page, heads_first, layout):
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(l)
    cache = mrsa.PagedKVCache(2, 40, hk, d, sequences=b + 2, max_len=160, page_size=page, dtype=dtype, device=dev)
    if heads_first:
        cache.pool = torch.empty(2, 2, 40, hk, page, d, dtype=dtype, device=dev).transpose(3, 4)
    cache.pool.zero_()
    seqs = torch.arange(b + 1, 1, -1, device=dev, dtype=torch.int32)
    cache.extend(seqs, torch.arange(b, device=dev, dtype=torch.int32) * 5 + l)
    x = torch.randn(b, l, hq + 2 * hk, d, device=dev, generator=g).to(dtype)
    q, k, v = x.split([hq, hk, hk], 2)
    inv = mrsa.rotary_inv_freq(2 * n, device=dev)[0] if n else None
    at = torch.arange(b, device=dev)[:, None] * 5 + torch.arange(l, device=dev)
    for pos in (None, (at * 2 + 1).contiguous()):
        y = cache.append(1, seqs, k, v, q=q if hq else None, inv_freq=inv, position_ids=pos if n else None,
                         attention_factor=1.25, layout=layout)
        cache.check()
        where = cache.table[seqs.long()[:, None], at // page].long()
        gk, gv = cache.pool[1, 0][where, at % page], cache.pool[1, 1][where, at % page]
        assert torch.equal(gv, v)
        if n:
            check_turned(gk, k, at if pos is None else pos, inv, 1.25, layout)
            check_turned(y, q, at if pos is None else pos, inv, 1.25, layout)
        else:
            assert torch.equal(gk, k) and y is None
    assert not cache.pool[0].any() and (cache.pool[1].ne(0).sum(-1).gt(0).sum() == 2 * b * l * hk)


@pytest.mark.gpu
def test_refusals(mrsa, cuda_device):
    dev = cuda_device
    cache = mrsa.PagedKVCache(1, 6, 2, 64, sequences=4, max_len=64, page_size=16, device=dev)
    k = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16, device=dev)
    s = cache.seqs(0)
    keep = torch.ones(1, 64, dtype=torch.bool, device=dev)
    state = cache.table, cache.lengths, cache.refcount
    for bad in [
        lambda: cache.free(s.long()), lambda: cache.free(s.cpu()), lambda: cache.free(s[None]),
        lambda: cache.free(torch.zeros(1025, dtype=torch.int32, device=dev)),
        lambda: cache.extend(s, -1), lambda: cache.extend(s, cache.seqs(1, 2)),
        lambda: cache.fork(s, cache.seqs(1, 2)), lambda: cache.fork(s, cache.seqs(1), cache.seqs(1, 2)),
        lambda: cache.compact(s, keep[:, :32]), lambda: cache.compact(s, keep.int()), lambda: cache.compact(s, keep.cpu()),
        lambda: mrsa.page_extend(*state, s, 1, page_size=48),
        lambda: mrsa.page_free(cache.table.t(), cache.lengths, cache.refcount, s),
        lambda: mrsa.page_free(cache.table, cache.lengths[:2], cache.refcount, s),
        lambda: mrsa.page_fork(cache.pool[:, :, :5], *state, s, cache.seqs(1)),
        lambda: mrsa.page_fork(cache.pool[..., :32], *state, s, cache.seqs(1)),
        lambda: mrsa.page_fork(cache.pool[0], *state, s, cache.seqs(1)),
        lambda: mrsa.page_copy(cache.pool, s, cache.seqs(1, 2)),
        lambda: cache.append(0, s, k, k[:, :, :1]), lambda: cache.append(0, s, k.float(), k.float()),
        lambda: cache.append(0, s, k[..., :32], k[..., :32]), lambda: cache.append(0, cache.seqs(0, 1), k, k),
        lambda: cache.append(0, s, k, k, layout="other"), lambda: cache.append(0, s, k, k, q=k[..., :32]),
        lambda: cache.append(0, s, k, k, start=cache.seqs(0, 0)),
        lambda: mrsa.PagedKVCache(1, 6, 2, 64, sequences=4, max_len=64, page_size=24, device=dev),
        lambda: mrsa.PagedKVCache(0, 6, 2, 64, sequences=4, max_len=64, device=dev),
    ]:
        with pytest.raises(ValueError):
            bad()
    cache.check()
    empty = cache.seqs()
    cache.free(empty), cache.extend(empty, 3), cache.fork(empty, empty), cache.compact(empty, keep[:0])


def test_page_argument_codes(mrsa):
    lib, L = mrsa._lib.load(), mrsa._lib
    P = 4096
    table = L.PAGE_TABLE.pack(P, P, P, 0, 4, 8, 100, 64)
    pool = L.PAGE_POOL.pack(P, 1, 2 << 20, 1 << 20, 64 * 512, 512, 256, 2, 256)
    size = lib.mrsa_page_workspace(table, 3)
    assert size > 0 and lib.mrsa_page_workspace(table, 1025) == 0 and lib.mrsa_page_workspace(None, 3) == 0
    assert lib.mrsa_page_free(None, P, 1, None) == L.ERR_NULL
    assert lib.mrsa_page_free(L.PAGE_TABLE.pack(P, P, 0, 0, 4, 8, 100, 64), P, 1, None) == L.ERR_NULL
    assert lib.mrsa_page_free(table, None, 1, None) == L.ERR_NULL
    assert lib.mrsa_page_free(table, P, 1025, None) == L.ERR_SHAPE and lib.mrsa_page_free(table, P, 0, None) == 0
    for ps in (0, 8, 24, 512):
        assert lib.mrsa_page_free(L.PAGE_TABLE.pack(P, P, P, 0, 4, 8, 100, ps), P, 1, None) == L.ERR_SHAPE
    assert lib.mrsa_page_extend(table, P, None, 1, 3, P, size - 1, None) == L.ERR_WORKSPACE
    assert lib.mrsa_page_extend(table, P, None, -1, 3, P, size, None) == L.ERR_ARG
    assert lib.mrsa_page_fork(table, None, P, P, None, 3, P, size, None) == L.ERR_NULL
    assert lib.mrsa_page_fork(table, pool, None, P, None, 3, P, size, None) == L.ERR_NULL
    bad = L.PAGE_POOL.pack(P, 1, 2 << 20, 1 << 20, 64 * 512, 1024, 256, 2, 256)      # tokens apart
    assert lib.mrsa_page_fork(table, bad, P, P, None, 3, P, size, None) == L.ERR_SHAPE
    bad = L.PAGE_POOL.pack(P + 8, 1, 2 << 20, 1 << 20, 64 * 512, 512, 256, 2, 256)
    assert lib.mrsa_page_fork(table, bad, P, P, None, 3, P, size, None) == L.ERR_ALIGN
    assert lib.mrsa_page_compact(table, pool, P, P + 1, 3, P, size, None) == L.ERR_ALIGN
    assert lib.mrsa_page_copy(table, pool, P, P, 101, None) == L.ERR_SHAPE
    assert lib.mrsa_page_copy(table, pool, None, P, 1, None) == L.ERR_NULL
    ra = L.ROTARY_ARGS.pack(0, 0, P, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 1, 0, 2, 128, 0, 1.0, 0, 0, 0)
    assert lib.mrsa_paged_append(ra, table, None, None) == L.ERR_NULL
    ap = L.APPEND_ARGS.pack(P, P, 0, P, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    assert lib.mrsa_paged_append(ra, table, ap, None) == L.ERR_NULL
    with pytest.raises(ValueError, match="CUDA"):
        mrsa.page_free(torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                       torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [2 ** 63 - 1, 2 ** 63 - 41, 2 ** 62, 2 ** 32, 2 ** 31 - 40])
def test_growth_past_any_whole_number_is_too_long(mrsa, cuda_device, tokens):
    """Sums with the lengths that pass 64 or 32 bits."""
    cache = mrsa.PagedKVCache(1, 12, 1, 64, sequences=3, max_len=128, page_size=16, device=cuda_device)
    cache.extend(cache.seqs(0, 1), 40)
    before = [cache.table.tolist(), cache.lengths.tolist(), cache.refcount.tolist()]
    for seqs in ((0,), (1, 0, 2), (2,)):
        cache.extend(cache.seqs(*seqs), tokens)
        with pytest.raises(ValueError, match="outgrow"):
            cache.check()
        assert [cache.table.tolist(), cache.lengths.tolist(), cache.refcount.tolist()] == before
    most = torch.tensor([2 ** 31 - 1], dtype=torch.int32, device=cuda_device)
    cache.extend(cache.seqs(0), most)
    with pytest.raises(ValueError, match="outgrow"):
        cache.check()
    with pytest.raises(OverflowError):
        cache.extend(cache.seqs(0), 2 ** 63)
    cache.extend(cache.seqs(0), 88)
    cache.check()
    assert cache.lengths.tolist() == [128, 40, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (80, torch.float16), (10, torch.float32)])
def test_append_of_the_same_tokens_twice(mrsa, cuda_device, d, dtype):
    """The first row of a batch that writes a token is carried out, a later one is not and is reported."""
    dev = cuda_device
    rows, l = 300, 3
    cache = mrsa.PagedKVCache(1, rows, 2, d, sequences=rows, max_len=16, page_size=16, dtype=dtype, device=dev)
    cache.extend(torch.arange(rows, dtype=torch.int32, device=dev), 12)
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(rows, l, 6, d, device=dev, generator=g).to(dtype)
    q, k, v = x.split([2, 2, 2], 2)

    def call(seqs, start=None):
        cache.pool.zero_()
        n = len(seqs)
        y = cache.append(0, cache.seqs(*seqs), k[:n], v[:n], q=q[:n], start=None if start is None else cache.seqs(*start))
        assert torch.equal(y, q[:n])                       # no frequencies: q as it is
        want = torch.zeros_like(cache.pool)
        done = []
        for i, s in enumerate(seqs):
            at = start[i] if start is not None else 12 - l
            if any(s == s2 and abs(at - at2) < l for s2, at2 in done):
                done.append((s, at))
                continue
            done.append((s, at))
            page = cache.table[s, 0]
            want[0, 0, page, at:at + l], want[0, 1, page, at:at + l] = k[i], v[i]
        assert torch.equal(cache.pool, want)

    def twice():
        with pytest.raises(ValueError, match="twice"):
            cache.check()

    call([4, 2, 4]), twice()
    call([7, 7]), twice()
    order = list(range(rows))
    call(order), cache.check()
    order[299] = 0
    call(order), twice()
    order[150] = 149
    call(order), twice()
    call([5, 5, 6], [0, 3, 0]), cache.check()              # neighbouring ranges of one sequence
    call([5, 5, 6], [0, 2, 2]), twice()
    call([5, 6, 5], [4, 2, 2]), twice()
    call([5, 5, 5, 5], [0, 9, 3, 6]), cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["tokens", "heads"])
def test_copies_that_depend_on_each_other(mrsa, cuda_device, layout):
    """All copies of a call are carried out, or none where two of them clash."""
    dev = cuda_device
    pages = 5000
    pool = torch.randint(-99, 99, (2, 2, pages, 16, 2, 16), device=dev).bfloat16()
    if layout == "heads":
        pool = pool.transpose(3, 4).contiguous().transpose(3, 4)
    status = torch.zeros(1, dtype=torch.int32, device=dev)

    def copy(src, dst, says):
        want = pool.clone()
        if not says & 32:
            ok = [(s, d) for s, d in zip(src, dst) if 0 <= s < pages and 0 <= d < pages]
            want[:, :, [d for _, d in ok]] = pool[:, :, [s for s, _ in ok]]
        status.zero_()
        t = [torch.tensor(x, dtype=torch.int32, device=dev) for x in (src, dst)]
        mrsa.page_copy(pool, *t, status=status)
        assert status.item() == says and torch.equal(pool, want)

    copy([1, 2], [3, 3], 32)                       # a target twice
    copy([1, 3], [3, 4], 32)                       # a target that is a source
    copy([1, 3], [3, 1], 32)                       # an exchange
    copy([1, 3, 9], [3, 5000, 9], 8)               # out of range, and a page onto itself: neither clashes
    copy([3, 4], [3, 3], 32)                       # a page that stays, and a copy to it
    copy([3, 3], [3, 4], 0)
    copy([7], [7], 0)
    copy([4, 4, 4], [5, 6, 7], 0)
    half = random.Random(1).sample(range(pages), pages)
    copy(half[:2500], half[2500:], 0)
    copy(half[:2500], half[2500:-1] + [half[2499]], 0)      # the last one onto itself
    copy(half[:2500], half[2500:-1] + [half[2498]], 32)
    copy(half[:2500], half[2500:-1] + [half[2500]], 32)


def test_checked_copy_argument_codes(mrsa):
    lib, L = mrsa._lib.load(), mrsa._lib
    P = 4096
    table = L.PAGE_TABLE.pack(P, P, P, 0, 4, 8, 100, 64)
    pool = L.PAGE_POOL.pack(P, 1, 2 << 20, 1 << 20, 64 * 512, 512, 256, 2, 256)
    size = lib.mrsa_page_copy_workspace(table)
    assert size >= 400 and lib.mrsa_page_copy_workspace(None) == 0
    assert lib.mrsa_page_copy_checked(None, pool, P, P, 2, P, size, None) == L.ERR_NULL
    assert lib.mrsa_page_copy_checked(table, pool, P, None, 2, P, size, None) == L.ERR_NULL
    assert lib.mrsa_page_copy_checked(table, pool, P, P, 101, P, size, None) == L.ERR_SHAPE
    assert lib.mrsa_page_copy_checked(table, pool, P, P, 2, P, size - 1, None) == L.ERR_WORKSPACE
    assert lib.mrsa_page_copy_checked(table, pool, P, P, 2, None, size, None) == L.ERR_WORKSPACE
    assert lib.mrsa_page_copy_checked(table, pool, P, P, 2, P + 4, size, None) == L.ERR_ALIGN
    assert lib.mrsa_page_copy_checked(table, pool, P, P, 0, None, 0, None) == 0


@pytest.mark.gpu
def test_pages_that_share_memory_are_refused(mrsa, cuda_device):
    dev = cuda_device
    cache = mrsa.PagedKVCache(2, 6, 2, 64, sequences=4, max_len=64, page_size=16, device=dev)
    s, pool = cache.seqs(0), cache.pool
    state = cache.table, cache.lengths
    cache.extend(s, 1)
    k = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16, device=dev)
    for dim, one in ((0, pool[:1]), (1, pool[:, :1]), (2, pool[:, :, :1]), (3, pool[:, :, :, :1])):
        same = one.expand(*[-1 if i != dim else pool.shape[dim] for i in range(6)])
        for bad in (lambda: mrsa.page_copy(same, s, cache.seqs(1)),
                    lambda: mrsa.page_fork(same, *state, cache.refcount, s, cache.seqs(1)),
                    lambda: mrsa.page_compact(same, *state, cache.refcount, s, torch.ones(1, 64, dtype=torch.bool, device=dev))):
            with pytest.raises(ValueError, match="share memory"):
                bad()
    kp, vp = pool[0]
    for pages in ((kp[:1].expand(6, -1, -1, -1), vp), (kp, vp[:, :1].expand(-1, 16, -1, -1)),
                  (kp, vp[:, :, :1].expand(-1, -1, 2, -1))):
        with pytest.raises(ValueError, match="share memory"):
            mrsa.paged_append(*pages, *state, s, k, k)
    with pytest.raises(ValueError, match="same memory"):
        mrsa.paged_append(kp, kp, *state, s, k, k)
    mrsa.paged_append(kp[:, :, ::2], vp[:, :, 1::2], *state, s, k[:, :, :1], k[:, :, :1])     # every second head: apart
    mrsa.paged_append(kp, vp, *state, s, k.expand(1, 1, 2, 64), k[:, :, :1].expand(1, 1, 2, 64))
    cache.check()
