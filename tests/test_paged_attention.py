"""Attention over pages (``paged_cache.paged_attention``) against the softmax
in 64 bits.

Bounds, before any run: with u the rounding of the type (2^-8 for bf16, 2^-11
for fp16, both twice the half ulp), an output is off by its own rounding, u |o|,
and by that of the probabilities where they enter the product in the type, at
most u sum p |v|; the scores' fp32 sums (128 products of O(1) numbers) move a
probability by 1e-5 of itself.  The LSE has the scores' error alone: 3e-5, and
1e-6 of itself."""

import math

import pytest
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def filled(mrsa, dev, lens, hkv, d, page, dtype, heads_first=False, seed=0, spare=3):
    """A cache of one layer whose sequences have these lengths on scattered pages; unused slots hold NaN."""
    g = torch.Generator(device=dev).manual_seed(seed)
    held = [-(-n // page) for n in lens]
    width, pages = max(1, max(held)), sum(held) + spare
    cache = mrsa.PagedKVCache(1, pages, hkv, d, sequences=len(lens), max_len=width * page, page_size=page, dtype=dtype,
                              device=dev)
    if heads_first:
        cache.pool = torch.empty(1, 2, pages, hkv, page, d, dtype=dtype, device=dev).transpose(3, 4)
    cache.pool.fill_(math.nan)
    order = torch.randperm(pages, device=dev, generator=g).tolist()
    for s, n in enumerate(lens):
        row, order = order[:held[s]], order[held[s]:]
        cache.table[s, :held[s]] = torch.tensor(row, dtype=torch.int32, device=dev)
        at = torch.arange(n, device=dev)
        where = torch.tensor(row, device=dev, dtype=torch.long)[at // page]
        cache.pool[0, :, where, at % page] = torch.randn(2, n, hkv, d, device=dev, generator=g).to(dtype)
    cache.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    return cache, g


def reference(cache, seqs, q, causal, valid, scale):
    """(o, sum p |v|, lse) in 64 bits."""
    b, l, hq, d = q.shape
    page, hkv = cache.page_size, cache.pool.shape[4]
    o = torch.zeros(b, l, hq, d, dtype=torch.float64, device=q.device)
    mass, lse = o.clone(), torch.full((b, l, hq), -math.inf, dtype=torch.float64, device=q.device)
    for i, s in enumerate(seqs.tolist()):
        n = cache.lengths[s].item()
        at = torch.arange(n, device=q.device)
        use = at if valid is None else at[valid[i, :n]]
        where = cache.table[s][use // page].long()
        k, v = cache.pool[0, :, where, use % page].double()          # [n, hkv, d]
        x = q[i].double().view(l, hkv, hq // hkv, d)
        z = torch.einsum("lhgd,nhd->lhgn", x, k) * scale
        if causal:
            late = use[None] > n - l + torch.arange(l, device=q.device)[:, None]
            z = z.masked_fill(late[:, None, None], -math.inf)
        if use.numel():
            lse[i] = torch.logsumexp(z, -1).view(l, hq)
            p = (z - lse[i].view(l, hkv, -1, 1)).exp().nan_to_num(0.0)
            o[i] = torch.einsum("lhgn,nhd->lhgd", p, v).reshape(l, hq, d)
            mass[i] = torch.einsum("lhgn,nhd->lhgd", p, v.abs()).reshape(l, hq, d)
    return o, mass, lse


def compare(mrsa, cache, seqs, q, causal=False, valid=None, scale=None):
    got, lse = cache.attend(0, seqs, q, causal=causal, key_valid=valid, scale=scale, return_lse=True)
    cache.check()
    want, mass, wlse = reference(cache, seqs, q, causal, valid, q.shape[-1] ** -0.5 if scale is None else scale)
    u = UNIT[q.dtype]
    assert got.dtype == q.dtype and got.shape == q.shape and lse.dtype == torch.float32
    err = (got.double() - want).abs()
    bound = u * want.abs() + (u + 1e-5) * mass + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
    assert (err <= bound).all(), (err / bound.clamp_min(1e-30)).max().item()
    empty = wlse == -math.inf
    assert torch.equal(lse == -math.inf, empty) and not got[empty].any()
    assert ((lse.double() - wlse)[~empty].abs() <= 3e-5 + 1e-6 * wlse[~empty].abs()).all()
    assert mrsa._lib.load().mrsa_device_error_flags(0) == 0
    return got, lse


def queries(dev, g, b, l, hq, d, dtype, strided=True):
    x = torch.randn(b, l, hq + (3 if strided else 0), d, device=dev, generator=g) * 1.5
    return x.to(dtype)[:, :, :hq]


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 127, 129, 700]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d,page,heads_first", [
    (28, 4, 128, 64, False), (2, 2, 64, 16, True), (12, 1, 128, 16, False), (20, 4, 64, 128, False),
    (16, 2, 128, 32, True), (40, 1, 64, 256, False)])
def test_one_token(mrsa, cuda_device, dtype, hq, hkv, d, page, heads_first):
    cache, g = filled(mrsa, cuda_device, LENS, hkv, d, page, dtype, heads_first)
    seqs = torch.randperm(len(LENS), device=cuda_device, generator=g).to(torch.int32)
    compare(mrsa, cache, seqs, queries(cuda_device, g, len(LENS), 1, hq, d, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("l,hq,hkv,d,page", [
    (2, 28, 4, 128, 64), (3, 5, 5, 128, 16), (5, 28, 4, 128, 64), (18, 7, 1, 128, 128), (19, 14, 2, 128, 32),
    (32, 28, 4, 128, 64), (37, 28, 4, 64, 16), (130, 6, 2, 64, 64), (33, 12, 1, 128, 256), (9, 24, 1, 64, 64)])
def test_blocks(mrsa, cuda_device, dtype, causal, l, hq, hkv, d, page):
    lens = [0, 1, 17, 64, 190, 700, 40]       # some shorter than the block: causal rows that see nothing
    cache, g = filled(mrsa, cuda_device, lens, hkv, d, page, dtype, seed=l)
    seqs = torch.tensor([6, 5, 4, 3, 2, 1, 0], dtype=torch.int32, device=cuda_device)
    compare(mrsa, cache, seqs, queries(cuda_device, g, len(lens), l, hq, d, dtype), causal)


@pytest.mark.gpu
@pytest.mark.parametrize("l", [1, 4, 32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_masks(mrsa, cuda_device, l, dtype):
    """Masked tokens that hold NaN and infinities, whole tiles and whole rows masked."""
    lens = [300, 129, 64, 200, 1, 77]
    cache, g = filled(mrsa, cuda_device, lens, 4, 128, 32, dtype, seed=9)
    width = cache.table.shape[1] * 32
    valid = torch.rand(len(lens), width, device=cuda_device, generator=g) < 0.5
    valid[1] = False                          # nothing left
    valid[2] = True
    valid[3, :160] = False                    # whole tiles
    valid[4] = False
    valid[5, 1:] = False                      # one token left
    valid[0, 0] = False
    seqs = torch.arange(len(lens), dtype=torch.int32, device=cuda_device)
    for s, n in enumerate(lens):
        at = torch.arange(n, device=cuda_device)[~valid[s, :n]]
        where = cache.table[s][at // 32].long()
        cache.pool[0, 0, where, at % 32] = math.inf
        cache.pool[0, 1, where, at % 32] = math.nan
    q = queries(cuda_device, g, len(lens), l, 28, 128, dtype)
    compare(mrsa, cache, seqs, q, False, valid)
    compare(mrsa, cache, seqs, q, True, valid)
    compare(mrsa, cache, seqs, q, False, torch.zeros_like(valid))


@pytest.mark.gpu
@pytest.mark.parametrize("l,dtype", [(1, torch.bfloat16), (32, torch.bfloat16), (32, torch.float16)])
def test_a_long_sequence_is_split(mrsa, cuda_device, l, dtype):
    cache, g = filled(mrsa, cuda_device, [40000, 3, 9001], 2, 128, 64, dtype, seed=2)
    seqs = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda_device)
    q = queries(cuda_device, g, 3, l, 14, 128, dtype)
    a = compare(mrsa, cache, seqs, q)
    b = cache.attend(0, seqs, q, return_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])     # the same bits every time


@pytest.mark.gpu
@pytest.mark.parametrize("l", [1, 32])
def test_extreme_scores(mrsa, cuda_device, l):
    """Scores that grow along the sequence (the running maximum moves all the time), and a token that takes all."""
    cache, g = filled(mrsa, cuda_device, [513], 1, 128, 64, torch.bfloat16, seed=4)
    at = torch.arange(513, device=cuda_device)
    where = cache.table[0][at // 64].long()
    q = torch.ones(1, l, 7, 128, dtype=torch.bfloat16, device=cuda_device)
    cache.pool[0, 0, where, at % 64] = (at / 64.0).bfloat16()[:, None, None]
    seqs = cache.seqs(0)
    compare(mrsa, cache, seqs, q, scale=2.0)
    compare(mrsa, cache, seqs, -q, scale=2.0)
    cache.pool[0, 0, cache.table[0, 3].long(), 5] = 30000.0
    compare(mrsa, cache, seqs, q, scale=1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("l", [1, 32])
def test_other_stream_and_many_rows(mrsa, cuda_device, l):
    lens = [((i * 37) % 90) for i in range(1100 if l == 1 else 70)]      # more rows than one launch takes
    cache, g = filled(mrsa, cuda_device, lens, 1, 64, 16, torch.bfloat16)
    seqs = torch.arange(len(lens), dtype=torch.int32, device=cuda_device)
    q = queries(cuda_device, g, len(lens), l, 3, 64, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        compare(mrsa, cache, seqs, q)


@pytest.mark.gpu
@pytest.mark.parametrize("l", [1, 32])
def test_bad_tables_are_reported(mrsa, cuda_device, l):
    cache, g = filled(mrsa, cuda_device, [100, 200], 4, 128, 64, torch.bfloat16)
    q = queries(cuda_device, g, 1, l, 28, 128, torch.bfloat16)
    for seq in (2, -1):
        o, lse = cache.attend(0, cache.seqs(seq), q, return_lse=True)
        with pytest.raises(ValueError, match="out of range"):
            cache.check()
        assert not o.any() and (lse == -math.inf).all()
    for bad in (-1, 10 ** 6):
        cache.table[1, 2] = bad                       # tokens 128 to 191 read as none
        o = cache.attend(0, cache.seqs(1), q)
        with pytest.raises(ValueError, match="lies outside"):
            cache.check()
        assert torch.isfinite(o).all()
    cache.lengths[0] = 10 ** 6
    assert not cache.attend(0, cache.seqs(0), q).any()
    with pytest.raises(ValueError, match="lies outside"):
        cache.check()


@pytest.mark.gpu
def test_refusals(mrsa, cuda_device):
    cache, g = filled(mrsa, cuda_device, [100], 4, 128, 64, torch.bfloat16)
    q = queries(cuda_device, g, 1, 1, 28, 128, torch.bfloat16)
    s = cache.seqs(0)
    valid = torch.ones(1, 128, dtype=torch.bool, device=cuda_device)
    k, v = cache.pool[0]
    state = cache.table, cache.lengths
    for bad in [
        lambda: cache.attend(0, s, q.float()), lambda: cache.attend(0, s, q.half()), lambda: cache.attend(0, s, q[0]),
        lambda: cache.attend(0, s, q[..., :64]), lambda: cache.attend(0, s, q[:, :, :27]),
        lambda: cache.attend(0, s, q[:, :, :2]), lambda: cache.attend(0, s, q.cpu()),
        lambda: cache.attend(0, cache.seqs(0, 0), q), lambda: cache.attend(0, s.long(), q),
        lambda: cache.attend(0, s, q, scale=0.0), lambda: cache.attend(0, s, q, scale=math.nan),
        lambda: cache.attend(0, s, q, key_valid=valid[:, :64]), lambda: cache.attend(0, s, q, key_valid=valid.int()),
        lambda: mrsa.paged_attention(q, k, v[:2], *state, s), lambda: mrsa.paged_attention(q, k, v.float(), *state, s),
        lambda: mrsa.paged_attention(q, k, v.transpose(2, 3), *state, s),
        lambda: mrsa.paged_attention(q, k[:, :48], v[:, :48], *state, s),
    ]:
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        cache.attend(0, s, q.clone().requires_grad_())
    none = torch.zeros(0, 1, 28, 128, dtype=torch.bfloat16, device=cuda_device)
    assert cache.attend(0, cache.seqs(), none).shape == none.shape
    assert cache.attend(0, s, q[:, :0]).shape == (1, 0, 28, 128)
    cache.check()


def test_argument_codes(mrsa):
    lib, L = mrsa._lib.load(), mrsa._lib
    P = 4096
    table = L.PAGE_TABLE.pack(P, P, 0, 0, 4, 8, 100, 64)

    def args(q=P, k=P, seqs=P, st=1024, b=1, l=1, hq=28, hkv=4, d=128, scale=0.1, dtype=0):
        return L.PAGED_ATTENTION_ARGS.pack(q, k, P, P, 0, 0, seqs, st, st, 128, 65536, 512, 128, 65536, 512, 128,
                                           b, l, hq, hkv, d, scale, dtype, 0)

    def rc(**kw):
        return lib.mrsa_paged_attention(args(**kw), table, None, 0, None)

    assert lib.mrsa_paged_attention(None, table, None, 0, None) == L.ERR_NULL
    assert lib.mrsa_paged_attention_workspace(None) == 0 and lib.mrsa_paged_attention_workspace(args(d=96)) == 0
    assert lib.mrsa_paged_attention_workspace(args()) > 0
    assert rc(q=0) == L.ERR_NULL and rc(k=0) == L.ERR_NULL and rc(seqs=0) == L.ERR_NULL
    assert rc(d=96) == L.ERR_SHAPE and rc(hq=27) == L.ERR_SHAPE and rc(hkv=0) == L.ERR_SHAPE and rc(b=-1) == L.ERR_SHAPE
    assert rc(scale=0.0) == L.ERR_ARG and rc(dtype=1) == L.ERR_ARG
    assert rc(q=P + 8) == L.ERR_ALIGN and rc(st=1025) == L.ERR_ALIGN
    assert rc() == L.ERR_WORKSPACE and rc(b=0) == 0 and rc(l=0) == 0
    bad = L.PAGE_TABLE.pack(P, P, 0, 0, 4, 8, 100, 48)
    assert lib.mrsa_paged_attention(args(), bad, None, 0, None) == L.ERR_SHAPE


@pytest.mark.gpu
@pytest.mark.parametrize("l,hq,hkv,d", [(1, 130, 1, 64), (2, 129, 1, 128), (1, 96, 1, 128), (1, 128, 1, 64), (64, 2, 1, 64),
                                        (128, 1, 1, 128), (129, 1, 1, 128), (43, 6, 2, 64)])
def test_groups_and_rows_at_the_tiles_edges(mrsa, cuda_device, l, hq, hkv, d):
    """Rows that fill an MMA tile, or miss it by one; more heads to a KV head than it has rows."""
    cache, g = filled(mrsa, cuda_device, [200, 0, 1, 3000, 130], hkv, d, 64, torch.bfloat16, seed=l + hq)
    seqs = torch.tensor([4, 3, 2, 1, 0], dtype=torch.int32, device=cuda_device)
    q = queries(cuda_device, g, 5, l, hq, d, torch.bfloat16)
    compare(mrsa, cache, seqs, q)
    compare(mrsa, cache, seqs, q, causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("l", [1, 32])
def test_strides(mrsa, cuda_device, l):
    """Every second head of the pages, a broadcast query, odd alignment, heads outside."""
    dev = cuda_device
    cache, g = filled(mrsa, dev, [150, 77], 4, 128, 32, torch.bfloat16)
    whole = cache.pool
    cache.pool = whole[:, :, :, :, ::2]
    seqs = cache.seqs(1, 0)
    compare(mrsa, cache, seqs, queries(dev, g, 1, l, 14, 128, torch.bfloat16).expand(2, l, 14, 128))
    flat = torch.randn(2 * l * 14 * 128 + 3, device=dev, generator=g).bfloat16()
    compare(mrsa, cache, seqs, flat[3:].view(2, l, 14, 128))
    compare(mrsa, cache, seqs, torch.randn(2, 14, l, 128, device=dev, generator=g).bfloat16().transpose(1, 2))
    with pytest.raises(ValueError, match="aligned"):
        cache.pool = torch.empty(2 * 9 * 32 * 2 * 128 + 1, device=dev, dtype=torch.bfloat16)[1:].view(1, 2, 9, 32, 2, 128)
        cache.attend(0, seqs, torch.zeros(2, l, 14, 128, device=dev, dtype=torch.bfloat16))


@pytest.mark.gpu
def test_offsets_past_32_bits(mrsa, cuda_device):
    """A pool of 4.7 GB a plane: the last pages and the first hold one sequence's tokens."""
    dev = cuda_device
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    g = torch.Generator(device=dev).manual_seed(1)
    pages = 36000
    cache = mrsa.PagedKVCache(1, pages, 8, 128, sequences=3, max_len=640, device=dev)
    assert cache.pool[0, 0].numel() * 2 > 1 << 32
    cache.refcount.fill_(1)                                   # only the ends are free
    cache.refcount[[3, 35990, 35999, 35991, 0, 35995, 35996, 35997, 5, 35998]] = 0
    cache.extend(cache.seqs(0), 300)
    assert cache.table[0, :5].tolist() == [0, 3, 5, 35990, 35991]
    k, v = torch.randn(2, 1, 300, 8, 128, device=dev, generator=g).bfloat16()
    cache.append(0, cache.seqs(0), k, v)
    cache.fork(cache.seqs(0), cache.seqs(1))
    keep = torch.ones(1, 640, dtype=torch.bool, device=dev)
    keep[0, 70:75] = False
    cache.compact(cache.seqs(1), keep)
    cache.check()
    assert cache.table[1, :5].tolist() == [0, 35996, 35997, 35998, 35999]
    for l, hq in ((1, 8), (32, 56)):
        compare(mrsa, cache, cache.seqs(1, 0), queries(dev, g, 2, l, hq, 128, torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d,page", [(28, 4, 128, 64), (5, 1, 64, 16), (32, 2, 128, 32)])
@pytest.mark.parametrize("lens", [[200], [511], [0, 130, 2048], [1, 64, 1985, 0]])
def test_few_short_sequences(mrsa, cuda_device, dtype, hq, hkv, d, page, lens):
    """One token of few sequences: several CTAs share a unit, some of them without a tile, or all masked."""
    cache, g = filled(mrsa, cuda_device, lens, hkv, d, page, dtype, seed=len(lens))
    seqs = torch.arange(len(lens), device=cuda_device, dtype=torch.int32).flip(0)
    q = queries(cuda_device, g, len(lens), 1, hq, d, dtype)
    first, lse = compare(mrsa, cache, seqs, q, causal=True)
    for _ in range(3):                        # the join has an order of its own: the same bits each time
        again, lse2 = cache.attend(0, seqs, q, causal=True, return_lse=True)
        assert torch.equal(first, again) and torch.equal(lse, lse2)
    width = cache.table.shape[1] * page
    valid = torch.rand(len(lens), width, device=cuda_device, generator=g) < 0.4
    valid[0] = False                          # a row that sees nothing
    valid[-1, :130] = False                   # leading shares that see nothing
    compare(mrsa, cache, seqs, q, valid=valid)


@pytest.mark.gpu
def test_flags_that_are_no_truth_value(mrsa, cuda_device):
    cache = mrsa.PagedKVCache(1, 6, 2, 64, sequences=4, max_len=64, page_size=16, device=cuda_device)
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16, device=cuda_device)
    two = torch.ones(2, dtype=torch.bool)
    for kw in (dict(causal=two), dict(return_lse=two)):
        with pytest.raises(RuntimeError, match="ambiguous"):
            cache.attend(0, cache.seqs(0), q, **kw)
    assert cache.attend(0, cache.seqs(0), q, causal=1, return_lse=0).shape == q.shape


def tight(got, lse, q, want, mass, wlse, weight, few):
    """Bounds for what the kernels promise, derived before any run.  The scores' fp32 sums move a probability by
    1e-5 of itself, in the product and in the sum that divides it; few rows: P in two 16-bit parts leaves 2^-17 of it
    (fp16: and, below its subnormals, 2^-25 of the maximum, with a sum of at least one), so 3e-5 of sum p |v| beside
    the output's own rounding, element by element.  Many rows: P is rounded once, independently per key, so the
    errors add in squares, those of one batch row's thousands of outputs to an rms of c of the root of o^2 + sum p^2 v^2.
    A rounding is off by u / m times a number uniform in [-1, 1], with a mantissa m whose logarithm is uniform in [1, 2):
    c = u / sqrt(3) sqrt(E[m^-2]) = 0.7355 u / sqrt(3); a factor of 1.2 for chance."""
    u = UNIT[q.dtype]
    err = (got.double() - want).abs()
    if few:
        bound = u * want.abs() + 3e-5 * mass + (2.0 ** -25 * (weight[1] + 1) if q.dtype == torch.float16 else 0.0)
        assert (err <= bound).all(), (err / bound.clamp_min(1e-30)).max().item()
    else:
        each = (1, 2, 3)
        rms = 0.7355 * u / math.sqrt(3) * (want.pow(2) + weight[0]).mean(each).sqrt() + 3e-5 * mass.mean(each)
        off = err.pow(2).mean(each).sqrt()
        assert (off <= 1.2 * rms).all(), (off / rms).tolist()
    seen = wlse > -math.inf
    assert ((lse.double() - wlse)[seen].abs() <= 3e-5 + 1e-6 * wlse[seen].abs()).all()


def weights(cache, seqs, q, valid=None):
    """Sums over the keys of (p v)^2 and of |v|, in 64 bits, [B, L, Hq, D]."""
    b, l, hq, d = q.shape
    page, hkv = cache.page_size, cache.pool.shape[4]
    squares = torch.zeros(b, l, hq, d, dtype=torch.float64, device=q.device)
    plain = squares.clone()
    for i, s in enumerate(seqs.tolist()):
        at = torch.arange(cache.lengths[s].item(), device=q.device)
        use = at if valid is None else at[valid[i, :at.numel()]]
        if use.numel():
            k, v = cache.pool[0, :, cache.table[s][use // page].long(), use % page].double()
            p = (torch.einsum("lhgd,nhd->lhgn", q[i].double().view(l, hkv, -1, d), k) * d ** -0.5).softmax(-1)
            squares[i] = torch.einsum("lhgn,nhd->lhgd", p * p, v * v).reshape(l, hq, d)
            plain[i] = v.abs().sum(0).repeat_interleave(hq // hkv, 0)
    return squares, plain


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", [[17, 64, 190, 700, 1, 333], [500], [9000, 100]])
@pytest.mark.parametrize("l,hq,hkv,d", [(1, 28, 4, 128), (2, 14, 2, 64), (1, 16, 1, 128), (4, 28, 4, 128), (32, 14, 2, 128),
                                        (40, 16, 2, 64)])
def test_no_more_than_the_stated_rounding(mrsa, cuda_device, l, hq, hkv, d, lens, dtype):
    cache, g = filled(mrsa, cuda_device, lens, hkv, d, 64, dtype, seed=l)
    seqs = torch.arange(len(lens), dtype=torch.int32, device=cuda_device)
    q = queries(cuda_device, g, len(lens), l, hq, d, dtype)
    valid = torch.rand(len(lens), cache.table.shape[1] * 64, device=cuda_device, generator=g) < 0.7
    for mask in (None, valid):
        got, lse = cache.attend(0, seqs, q, key_valid=mask, return_lse=True)
        cache.check()
        tight(got, lse, q, *reference(cache, seqs, q, False, mask, d ** -0.5), weights(cache, seqs, q, mask),
              l * (hq // hkv) <= 16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("l,page", [(1, 64), (2, 16), (4, 128), (32, 64), (45, 32)])
def test_every_tile_has_its_own_values(mrsa, cuda_device, l, page, dtype):
    """Each query looks at one 64-key tile of a long sequence, whose keys and values are that tile's alone: a tile
    read, weighed or joined in another's place is off by all of the output."""
    dev = cuda_device
    lens = [40000, 6401]
    cache, g = filled(mrsa, dev, lens, 2, 128, page, dtype, seed=l)
    tiles = [-(-n // 64) for n in lens]
    code = torch.randint(0, 2, (sum(tiles), 2, 128), device=dev, generator=g).to(dtype) * 2 - 1
    value = torch.randn(sum(tiles), 2, 128, device=dev, generator=g).to(dtype)
    for s, n in enumerate(lens):
        at = torch.arange(n, device=dev)
        tile = at // 64 + sum(tiles[:s])
        where = cache.table[s][at // page].long()
        cache.pool[0, 0, where, at % page], cache.pool[0, 1, where, at % page] = code[tile], value[tile]
    seqs = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    for turn in range(4 if l > 2 else 12):
        q = torch.empty(2, l, 14, 128, dtype=dtype, device=dev)
        want = torch.empty_like(q, dtype=torch.float64)
        for s in range(2):
            pick = sum(tiles[:s]) + torch.randint(0, tiles[s], (l, 2, 7), device=dev, generator=g)
            pick[0, :, 0], pick[0, :, 1] = sum(tiles[:s]), sum(tiles[:s + 1]) - 1        # the first and the last
            heads = torch.arange(2, device=dev)[None, :, None]
            q[s] = (2 * code[pick, heads]).view(l, 14, 128)
            want[s] = value[pick, heads].double().view(l, 14, 128)
        got, lse = compare(mrsa, cache, seqs, q)
        # the tile that is looked at has a score of 22.6, the others' are normal around 0 with a deviation of 2
        assert ((got.double() - want).abs() <= 3 * UNIT[dtype] * want.abs() + 1e-3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("width", [4, 40])
@pytest.mark.parametrize("l", [1, 2, 4, 32])
def test_pages_out_of_range_read_as_masked(mrsa, cuda_device, l, width):
    cache, g = filled(mrsa, cuda_device, [100, 200], 4, 128, 64, torch.bfloat16)
    cache.table = torch.cat((cache.table, cache.table.new_full((2, width - 4), -1)), 1).contiguous()
    q = queries(cuda_device, g, 1, l, 28, 128, torch.bfloat16)
    seqs, page = cache.seqs(1), cache.table[1, 2].clone()
    valid = torch.ones(1, width * 64, dtype=torch.bool, device=cuda_device)
    valid[0, 128:192] = False
    want, mass, wlse = reference(cache, seqs, q, False, valid, 128 ** -0.5)
    for bad in (-1, 10 ** 6):
        cache.table[1, 2] = bad
        o, lse = cache.attend(0, seqs, q, return_lse=True)
        with pytest.raises(ValueError, match="lies outside"):
            cache.check()
        cache.table[1, 2] = page
        u = UNIT[torch.bfloat16]
        assert ((o.double() - want).abs() <= u * want.abs() + (u + 1e-5) * mass).all()
        assert ((lse.double() - wlse).abs() <= 3e-5 + 1e-6 * wlse.abs()).all()
