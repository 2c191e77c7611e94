"""What the rotary and paged operators do not differentiate they refuse: a
gradient or a tangent is never lost without an error."""

import pytest
import torch


def append_args(mrsa, dev):
    cache = mrsa.PagedKVCache(1, 6, 2, 64, sequences=4, max_len=64, page_size=16, device=dev)
    cache.extend(cache.seqs(0), 3)
    g = torch.Generator(device=dev).manual_seed(1)
    q, k, v = torch.randn(1, 3, 8, 64, device=dev, generator=g).bfloat16().split([4, 2, 2], 2)
    return cache, dict(q=q.clone(), k=k.clone(), v=v.clone(), k_pages=cache.pool[0, 0], v_pages=cache.pool[0, 1],
                       inv_freq=mrsa.rotary_inv_freq(64, device=dev)[0])


def append(mrsa, cache, a):
    return mrsa.paged_append(a["k_pages"], a["v_pages"], cache.table, cache.lengths, cache.seqs(0), a["k"], a["v"],
                             q=a["q"], inv_freq=a["inv_freq"], status=cache.status)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["q", "k", "v", "k_pages", "v_pages"])
def test_append_refuses_a_gradient(mrsa, cuda_device, name):
    """Forward only: a gradient that would be lost is an error, and nothing is written."""
    cache, a = append_args(mrsa, cuda_device)
    cache.pool.zero_()
    a[name] = a[name].detach().requires_grad_()
    with pytest.raises(NotImplementedError, match="forward-only"):
        append(mrsa, cache, a)
    assert not cache.pool.any()
    with torch.no_grad():
        append(mrsa, cache, a)
    cache.check()
    assert cache.pool.any()


@pytest.mark.gpu
def test_tangents_are_refused(mrsa, cuda_device):
    from torch.autograd import forward_ad

    cache, a = append_args(mrsa, cuda_device)
    pos = torch.arange(3, device=cuda_device)[None]
    state = cache.table, cache.lengths, cache.seqs(0)
    calls = {
        "rotary": (("q", "k", "inv_freq"), lambda a: mrsa.rotary_embedding(a["q"], a["k"], pos, a["inv_freq"])),
        "append": (("q", "k", "v", "k_pages", "v_pages", "inv_freq"), lambda a: append(mrsa, cache, a)),
        "attend": (("q", "k_pages", "v_pages"), lambda a: mrsa.paged_attention(a["q"], a["k_pages"], a["v_pages"], *state)),
    }
    with forward_ad.dual_level():
        for names, call in calls.values():
            for name in names:
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(a | {name: forward_ad.make_dual(a[name], torch.ones_like(a[name]))})
            with torch.no_grad():
                call(a)


@pytest.mark.gpu
def test_gradient_of_frequencies_is_refused(mrsa, cuda_device):
    cache, a = append_args(mrsa, cuda_device)
    pos = torch.arange(3, device=cuda_device)[None]
    inv = a["inv_freq"].requires_grad_()
    for wants in (False, True):
        q = a["q"].detach().requires_grad_(wants)
        with pytest.raises(NotImplementedError, match="inv_freq"):
            mrsa.rotary_embedding(q, a["k"], pos, inv)
    with pytest.raises(NotImplementedError, match="inv_freq"):
        append(mrsa, cache, a)
    with torch.no_grad():
        y, _ = mrsa.rotary_embedding(a["q"], a["k"], pos, inv)
        assert torch.equal(append(mrsa, cache, a), y)
