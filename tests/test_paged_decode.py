"""Block decoding over pages (``paged_decode.py``): prefill, candidates, a
thinned prompt, against the same model in plain fp32 torch with lists for a
cache.  The logits have a cosine similarity above 0.999 (bf16 layers on one
side), as for the routed model in ``test_gpu_dream.py``; what has to be the
same call is the same bit for bit."""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


class Plain:
    """The model in fp32; `cache[layer]` is (k, v) of one sequence, [n, heads, d]."""

    def __init__(self, model):
        self.m = model
        self.cache = [None] * model.cfg.layers

    def step(self, ids, pos, over=0, causal=False):
        """Tokens appended, after the last `over` of the cache were dropped."""
        m, c = self.m, self.m.cfg
        x = m.embed[ids].float()
        ang = pos.float()[:, None] * m.inv_freq
        cos, sin = (t(ang)[:, None] * m.attention_factor for t in (torch.cos, torch.sin))

        def turn(t):
            a, b = t.chunk(2, -1)
            return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

        def norm(t):
            return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + c.rms_eps)

        n = ids.shape[0]
        for i in range(c.layers):
            lay = {k: t.float() for k, t in m.layers[i].items() if torch.is_tensor(t)}
            wg, wu = (w.float() for w in m.gate_up(i))
            h = norm(x)
            q = turn((h @ lay["wq"].T).view(n, c.q_heads, c.head_dim))
            k = turn((h @ lay["wk"].T).view(n, c.kv_heads, c.head_dim))
            v = (h @ lay["wv"].T).view(n, c.kv_heads, c.head_dim)
            if self.cache[i] is not None:
                k0, v0 = (t[:t.shape[0] - over] for t in self.cache[i])
                k, v = torch.cat((k0, k)), torch.cat((v0, v))
            self.cache[i] = (k, v)
            g = c.q_heads // c.kv_heads
            s = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(g, 1)) * c.head_dim ** -0.5
            if causal:
                late = torch.arange(k.shape[0], device=x.device) > k.shape[0] - n + torch.arange(n, device=x.device)[:, None]
                s = s.masked_fill(late, float("-inf"))
            o = torch.einsum("hqk,khd->qhd", s.softmax(-1), v.repeat_interleave(g, 1)).reshape(n, -1)
            x = x + o @ lay["wo"].T
            h = norm(x)
            x = x + (F.silu(h @ wg.T) * (h @ wu.T)) @ lay["wd"].T
        return norm(x) @ m.lm_head.float().T


def close(got, want):
    assert torch.isfinite(got).all()
    cos = F.cosine_similarity(got.float().flatten(), want.flatten(), dim=0)
    assert cos > 0.999, float(cos)


@pytest.fixture(scope="module")
def decoder(mrsa, cuda_device):
    from mrsa_b200.dream_forward import DreamConfig, DreamForward
    from mrsa_b200.paged_decode import PagedDream

    cfg = DreamConfig(layers=2, hidden=896, ffn=1024, q_heads=14, kv_heads=2, vocab=512)
    return PagedDream(DreamForward(cfg, seed=3, device=cuda_device), pages=64, sequences=6, max_len=640)


def test_candidates_of_one_prompt(decoder, cuda_device):
    dec, cache = decoder, decoder.cache
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(1)
    prompt = torch.randint(0, 512, (1, 203), device=dev, generator=g)
    blocks = torch.randint(0, 512, (2, 3, 32), device=dev, generator=g)
    at = torch.arange(640, device=dev)
    cache.free(cache.seqs(*range(6)))
    seq, cands = cache.seqs(4), cache.seqs(0, 5, 2)
    plain = Plain(dec.model)
    close(dec.prefill(seq, prompt)[0], plain.step(prompt[0], at[:203]))
    used = (cache.refcount > 0).sum().item()
    dec.fork(seq, cands)
    assert (cache.refcount > 0).sum().item() == used + 3          # three whole pages in common, the fourth copied
    cache.extend(cands, 32)
    kept = list(plain.cache)
    first = dec.step(cands, blocks[0])
    second = dec.step(cands, blocks[1])                           # the block rewritten
    cache.check()
    for i in range(3):
        plain.cache = list(kept)
        close(first[i], plain.step(blocks[0, i], at[203:235]))
        close(second[i], plain.step(blocks[1, i], at[203:235], over=32))
    # the prompt itself was not touched: a later candidate of it gives the same bits
    late = cache.seqs(1)
    dec.fork(seq, late)
    cache.extend(late, 32)
    again = dec.step(late, blocks[0, :1])
    alone = dec.step(cache.seqs(0), blocks[0, :1])
    cache.check()
    assert torch.equal(again, alone)
    cache.free(cands)
    cache.free(late)
    cache.free(seq)
    cache.check()
    assert not cache.refcount.any() and (cache.table == -1).all()


def test_tokens_one_by_one_and_a_thinned_prompt(decoder, cuda_device):
    dec, cache = decoder, decoder.cache
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(2)
    prompt = torch.randint(0, 512, (1, 300), device=dev, generator=g)
    new = torch.randint(0, 512, (1, 4), device=dev, generator=g)
    at = torch.arange(640, device=dev)
    cache.free(cache.seqs(*range(6)))
    seq, thin = cache.seqs(3), cache.seqs(1)
    plain = Plain(dec.model)
    close(dec.prefill(seq, prompt, causal=True)[0], plain.step(prompt[0], at[:300], causal=True))
    dec.fork(seq, thin)
    keep = torch.rand(1, 640, device=dev, generator=g) < 0.6
    keep[0, :70] = True
    cache.compact(thin, keep)
    few = Plain(dec.model)
    few.cache = [tuple(t[keep[0, :300]] for t in kv) for kv in plain.cache]
    left = int(keep[0, :300].sum())
    for i in range(4):
        pos = at[None, 300 + i:301 + i].contiguous()
        close(dec.prefill(seq, new[:, i:i + 1], causal=True)[0], plain.step(new[0, i:i + 1], pos[0]))
        # the thinned copy keeps its tokens' positions
        close(dec.prefill(thin, new[:, i:i + 1], position_ids=pos)[0], few.step(new[0, i:i + 1], pos[0]))
    cache.check()
    assert cache.lengths[cache.seqs(3, 1).long()].tolist() == [304, left + 4]


@pytest.mark.parametrize("pages,max_len,causal,error", [(4, 640, False, RuntimeError), (4, 640, True, RuntimeError),
                                                        (9, 256, False, ValueError)])
def test_prefill_without_room_keeps_what_is_cached(mrsa, cuda_device, pages, max_len, causal, error):
    from mrsa_b200.dream_forward import DreamConfig, DreamForward
    from mrsa_b200.paged_decode import PagedDream

    dev = cuda_device
    cfg = DreamConfig(layers=2, hidden=896, ffn=1024, q_heads=14, kv_heads=2, vocab=512)
    dec = PagedDream(DreamForward(cfg, seed=3, device=dev), pages=pages, sequences=2, max_len=max_len)
    cache = dec.cache
    ids = torch.randint(0, 512, (1, 300), device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    dec.prefill(cache.seqs(1), ids[:, :200], causal=causal)
    cache.check()
    state = [t.clone() for t in (cache.pool.view(torch.int16), cache.table, cache.lengths, cache.refcount)]
    dec.prefill(cache.seqs(1), ids[:, 200:], causal=causal)        # 300 tokens need five pages
    with pytest.raises(error):
        cache.check()
    for was, now in zip(state, (cache.pool.view(torch.int16), cache.table, cache.lengths, cache.refcount)):
        assert torch.equal(was, now)
    dec.prefill(cache.seqs(5), ids[:, :7])                         # no such sequence
    with pytest.raises(ValueError, match="out of range"):
        cache.check()
    # what fits still continues the same tokens
    a = dec.prefill(cache.seqs(1), ids[:, 200:250], causal=causal)
    cache.check()
    cache.free(cache.seqs(1))
    dec.prefill(cache.seqs(0), ids[:, :200], causal=causal)
    b = dec.prefill(cache.seqs(0), ids[:, 200:250], causal=causal)
    cache.check()
    assert torch.equal(a, b)
