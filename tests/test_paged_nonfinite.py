"""Scores that are not finite in attention over pages: a query that sees a NaN
or a score of +infinity has no softmax, so its output is NaN and its LSE is no
number below infinity; one of -infinity is a weight of zero; a query that sees
nothing still gets zeros and -infinity, whatever it holds itself.  The other
rows keep the bounds of ``test_paged_attention.py``."""

import math

import pytest
import torch

from test_paged_attention import UNIT, filled, queries, reference

# lengths and table width in tokens: whole units, clusters of CTAs (one token of
# few sequences), stretches that end inside a unit
FORMS = {"whole": ([150, 190, 65, 1, 130, 177], 0), "cluster": ([500], 0), "cut": ([700, 150], 4096)}


def wide(cache, tokens):
    """The table with room for `tokens` per sequence."""
    more = tokens // cache.page_size - cache.table.shape[1]
    if more > 0:
        cache.table = torch.cat((cache.table, cache.table.new_full((cache.table.shape[0], more), -1)), 1).contiguous()


def scores(cache, seqs, q, causal, valid):
    """Whether a row sees a score that is NaN or +infinity, [B, L, Hq]."""
    b, l, hq, d = q.shape
    page, hkv = cache.page_size, cache.pool.shape[4]
    bad = torch.zeros(b, l, hq, dtype=torch.bool, device=q.device)
    for i, s in enumerate(seqs.tolist()):
        n = cache.lengths[s].item()
        at = torch.arange(n, device=q.device)
        use = at if valid is None else at[valid[i, :n]]
        k = cache.pool[0, 0, cache.table[s][use // page].long(), use % page].double()
        z = torch.einsum("lhgd,nhd->lhgn", q[i].double().view(l, hkv, hq // hkv, d), k)
        wrong = z.isnan() | (z == math.inf)
        if causal:
            wrong &= (use[None] <= n - l + torch.arange(l, device=q.device)[:, None])[:, None, None]
        bad[i] = wrong.any(-1).view(l, hq)
    return bad


def compare(mrsa, cache, seqs, q, causal=False, valid=None):
    got, lse = cache.attend(0, seqs, q, causal=causal, key_valid=valid, return_lse=True)
    cache.check()
    bad = scores(cache, seqs, q, causal, valid)
    want, mass, wlse = reference(cache, seqs, q, causal, valid, q.shape[-1] ** -0.5)
    assert got[bad].isnan().all() and not lse[bad].isfinite().any() and not (lse[bad] == -math.inf).any()
    u = UNIT[q.dtype]
    err = (got.double() - want).abs()[~bad]
    assert (err <= (u * want.abs() + (u + 1e-5) * mass)[~bad] + 2.0 ** -25).all()
    empty = (wlse == -math.inf) & ~bad
    assert torch.equal((lse == -math.inf) & ~bad, empty) and not got[empty].any()
    fine = ~bad & ~empty
    assert ((lse.double() - wlse)[fine].abs() <= 3e-5 + 1e-6 * wlse[fine].abs()).all()
    assert mrsa._lib.load().mrsa_device_error_flags(0) == 0
    return bad


def spoil(mrsa, dev, l, form, dtype):
    lens, tokens = FORMS[form]
    cache, g = filled(mrsa, dev, lens, 4, 128, 64, dtype, seed=l)
    wide(cache, tokens)
    seqs = torch.arange(len(lens), dtype=torch.int32, device=dev)
    q = queries(dev, g, len(lens), l, 28, 128, dtype, strided=False)
    keys = cache.pool[0, 0]
    page = cache.table[0].long()
    sound = keys.clone()
    # a NaN in one key of one head, at each of eight neighbouring slots
    for slot in range(72, 80):
        keys[page[slot // 64], slot % 64, 1, 5] = math.nan
        assert compare(mrsa, cache, seqs, q)[0].sum() == 7 * l
        keys.copy_(sound)
    # a score of +infinity where q is above zero, of -infinity where it is below
    for slot in range(72, 80):
        keys[page[slot // 64], slot % 64, 2, 0] = math.inf
        bad = compare(mrsa, cache, seqs, q)
        assert torch.equal(bad[0, :, 14:21], q[0, :, 14:21, 0] >= 0)
        keys.copy_(sound)
    # nothing but NaN, nothing but -infinity
    keys[page[page >= 0], :, 3] = math.nan
    assert compare(mrsa, cache, seqs, q)[0].sum() == 7 * l
    q0 = q.clone()
    q0[0, :, 21:, 0] = -1.0
    keys.copy_(sound)
    keys[page[page >= 0], :, 3, 0] = math.inf
    assert not compare(mrsa, cache, seqs, q0)[0].any()
    keys.copy_(sound)
    # a NaN and infinities in q: its own row alone
    q1 = q.clone()
    q1[0, l - 1, 4, 9] = math.nan
    q1[-1, 0, 20, 100] = math.inf
    bad = compare(mrsa, cache, seqs, q1)
    assert bad.sum() == 2
    compare(mrsa, cache, seqs, q1, causal=True)
    # rows that see nothing
    valid = torch.ones(len(lens), cache.table.shape[1] * 64, dtype=torch.bool, device=dev)
    valid[0] = False
    compare(mrsa, cache, seqs, q1, valid=valid)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("l", [1, 2])
def test_few_rows_keep_what_is_not_finite(mrsa, cuda_device, l, form, dtype):
    spoil(mrsa, cuda_device, l, form, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("l", [4, 16, 32, 45])
def test_many_rows_keep_what_is_not_finite(mrsa, cuda_device, l, form, dtype):
    spoil(mrsa, cuda_device, l, form, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["whole", "cut"])
@pytest.mark.parametrize("l", [2, 32])
def test_rows_before_the_cache_get_zeros(mrsa, cuda_device, l, form):
    """Causal queries that see nothing, of a sequence whose every value is NaN."""
    cache, g = filled(mrsa, cuda_device, [1], 4, 128, 64, torch.bfloat16)
    wide(cache, FORMS[form][1])
    cache.pool[0, 1] = math.nan
    o, lse = cache.attend(0, cache.seqs(0), queries(cuda_device, g, 1, l, 28, 128, torch.bfloat16), causal=True,
                          return_lse=True)
    cache.check()
    assert not o[0, :-1].any() and (lse[0, :-1] == -math.inf).all() and o[0, -1].isnan().all()
