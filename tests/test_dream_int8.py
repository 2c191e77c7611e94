"""The Dream-shaped model with dense layers in 8 bits (``dream_int8.py``).

Against fp32 with the weights that the whole numbers stand for: what differs is
the activations' quantization.  A row whose largest value is m times its root
mean square is off by m / 127 / sqrt(12) of itself: 0.8 % for a normal row of a
thousand (m = 3.5), 2.3 % behind the gate (m = 10), and no more than 6 % in the
logits of two layers, a cosine above 0.998.  What has to be the same call is the
same bit for bit."""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def values(w):
    return w[0].float() * w[1][:, None]


class Plain:
    """One sequence in fp32, every token seeing all, its keys and values kept."""

    def __init__(self, m):
        self.m, self.cache = m, [None] * m.cfg.layers

    def step(self, ids, pos):
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
        for i, lay in enumerate(m.layers):
            qkv = (norm(x) @ values(lay["wqkv"]).T + lay["bqkv"].float()).view(n, -1, c.head_dim)
            q, k, v = torch.split(qkv, (c.q_heads, c.kv_heads, c.kv_heads), dim=1)
            q, k = turn(q), turn(k)
            if self.cache[i] is not None:
                k, v = torch.cat((self.cache[i][0], k)), torch.cat((self.cache[i][1], v))
            self.cache[i] = k, v
            g = c.q_heads // c.kv_heads
            s = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(g, 1)) * c.head_dim ** -0.5
            o = torch.einsum("hqk,khd->qhd", s.softmax(-1), v.repeat_interleave(g, 1)).reshape(n, -1)
            x = x + o @ values(lay["wo"]).T
            h = norm(x)
            wg, wu = m.gate_up(i)
            x = x + (F.silu(h @ wg.T) * (h @ wu.T)) @ values(lay["wd"]).T
        return norm(x) @ values(m.lm_head).T


def close(got, want):
    assert torch.isfinite(got).all()
    cos = F.cosine_similarity(got.float().flatten(), want.flatten(), dim=0)
    assert cos > 0.998, float(cos)


@pytest.fixture(scope="module")
def models(mrsa, cuda_device):
    from mrsa_b200.dream_forward import DreamConfig, DreamForward

    cfg = DreamConfig(layers=4, hidden=896, ffn=1024, q_heads=7, kv_heads=1, vocab=520, swa_window=300)
    model = DreamForward(cfg, seed=3, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(4)
    for lay in model.layers:
        for k in ("bq", "bk", "bv"):
            lay[k] = torch.randn(lay[k].shape, device=cuda_device, generator=g).bfloat16() * 0.1
    return model, mrsa.DreamInt8(model)


def test_block_decoding(models, cuda_device):
    from mrsa_b200.paged_decode import PagedDream

    dev, m = cuda_device, models[1]
    dec = PagedDream(m, pages=64, sequences=6, max_len=512)
    g = torch.Generator(device=dev).manual_seed(1)
    prompt = torch.randint(0, 520, (1, 203), device=dev, generator=g)
    blocks = torch.randint(0, 520, (3, 32), device=dev, generator=g)
    at = torch.arange(512, device=dev)
    cache, seq, cands = dec.cache, dec.cache.seqs(4), dec.cache.seqs(0, 5, 2)
    plain = Plain(m)
    close(dec.prefill(seq, prompt)[0], plain.step(prompt[0], at[:203]))
    dec.fork(seq, cands)
    cache.extend(cands, 32)
    got = dec.step(cands, blocks)
    again = dec.step(cands, blocks)
    cache.check()
    assert torch.equal(got, again)
    kept = list(plain.cache)
    for i in range(3):
        plain.cache = list(kept)
        close(got[i], plain.step(blocks[i], at[203:235]))
    # a candidate by itself, and one token after the other
    late = cache.seqs(1)
    dec.fork(seq, late)
    cache.extend(late, 32)
    assert torch.equal(dec.step(late, blocks[:1]), dec.step(cache.seqs(0), blocks[:1]))
    one = dec.prefill(late, blocks[:1, :1])
    assert one.shape == (1, 1, 520) and torch.isfinite(one).all()
    hidden = dec.step(cands, blocks, logits=False)
    assert hidden.shape == (3, 32, 896) and hidden.dtype == torch.bfloat16
    cache.check()


def test_forward_with_route_layers(models, mrsa, cuda_device):
    """The whole forward (three window layers and a routed one) against its steps by the public operators, bit for
    bit, and near the bf16 model."""
    from mrsa_b200.dream_forward import landmark_inputs

    model, m = models
    c = m.cfg
    ids, pos, lmk = landmark_inputs(1, 512, c, mask_id=c.vocab - 1, device=cuda_device)
    logits, xs = m(ids, pos, return_layer_inputs=True)
    assert logits.shape == (1, 512, c.vocab) and len(xs) == 4 and xs[1].shape == (1, 512, c.hidden)
    with torch.inference_mode():
        x, delta = None, torch.where(lmk[None, :, None], m.embed[ids] + m.role, m.embed[ids])
        for i, lay in enumerate(m.layers):
            h = None
            if c.is_route(i):
                h, x = mrsa.add_rms_norm(delta, x, lay["in_norm"], c.rms_eps)
                q8, s8 = mrsa.quantize_int8(h)
            else:
                q8, s8, x = mrsa.add_rms_norm_int8(delta, x, lay["in_norm"], c.rms_eps)
            assert torch.equal(x, xs[i])
            qkv = mrsa.linear_int8(q8, s8, *lay["wqkv"], lay["bqkv"]).view(1, 512, 9, 128)
            o = m.attend(i, qkv[:, :, :7], qkv[:, :, 7:8], qkv[:, :, 8:], h, pos, None)
            delta = mrsa.linear_int8(*mrsa.quantize_int8(o), *lay["wo"])
            q8, s8, x = mrsa.add_rms_norm_int8(delta, x, lay["post_norm"], c.rms_eps)
            delta = mrsa.linear_int8(*mrsa.quantize_int8(mrsa.swiglu_int8(q8, s8, *lay["wgu"])), *lay["wd"])
        q8, s8, _ = mrsa.add_rms_norm_int8(delta, x, m.final_norm, c.rms_eps)
        assert torch.equal(mrsa.linear_int8(q8, s8, *m.lm_head), logits)
    hidden = m(ids, pos, logits=False)
    assert torch.equal(hidden, mrsa.add_rms_norm(delta, x, m.final_norm, c.rms_eps)[0])
    # weights too are off by 0.8 %; routing that flips moves single rows further
    cos = F.cosine_similarity(logits.float().flatten(), model(ids, pos).float().flatten(), dim=0)
    assert cos > 0.99, float(cos)
    assert "wq" not in m.layers[0] and m.embed is model.embed


def test_norm_weights_by_layer(mrsa, cuda_device):
    """Norm weights of their own for every norm: each where it belongs, in the forward and over pages."""
    from mrsa_b200.dream_forward import DreamConfig, DreamForward
    from mrsa_b200.paged_decode import PagedDream

    dev = cuda_device
    cfg = DreamConfig(layers=4, hidden=896, ffn=1024, q_heads=7, kv_heads=1, vocab=520, swa_window=300)
    model = DreamForward(cfg, seed=5, device=dev)
    g = torch.Generator(device=dev).manual_seed(6)
    for where, k in [(lay, k) for lay in model.layers for k in ("in_norm", "post_norm")] + [(vars(model), "final_norm")]:
        where[k] = (torch.rand(cfg.hidden, device=dev, generator=g) * 2 + 0.2).bfloat16()
    m = mrsa.DreamInt8(model)
    ids = torch.randint(0, 520, (1, 512), device=dev, generator=g)
    pos = torch.arange(512, device=dev)[None]
    lmk = (pos[0] + 1) % cfg.chunk == 0

    def layer(i, delta, x, attention):
        """The layer by the public operators; attention(q, k, v, normed input)."""
        h, x = mrsa.add_rms_norm(delta, x, model.layers[i]["in_norm"], cfg.rms_eps)
        q8 = mrsa.quantize_int8(h) if "route" in model.layers[i] else None
        if q8 is None:
            q8 = mrsa.add_rms_norm_int8(x, None, model.layers[i]["in_norm"], cfg.rms_eps)[:2]
        qkv = mrsa.linear_int8(*q8, *m.layers[i]["wqkv"], m.layers[i]["bqkv"]).view(1, 512, 9, 128)
        o = attention(i, qkv[:, :, :7], qkv[:, :, 7:8], qkv[:, :, 8:], h)
        delta = mrsa.linear_int8(*mrsa.quantize_int8(o), *m.layers[i]["wo"])
        q8, s8, x = mrsa.add_rms_norm_int8(delta, x, model.layers[i]["post_norm"], cfg.rms_eps)
        return mrsa.linear_int8(*mrsa.quantize_int8(mrsa.swiglu_int8(q8, s8, *m.layers[i]["wgu"])), *m.layers[i]["wd"]), x

    def model_by(first, attention):
        delta, x = first, None
        for i in range(cfg.layers):
            delta, x = layer(i, delta, x, attention)
        q8, s8, _ = mrsa.add_rms_norm_int8(delta, x, model.final_norm, cfg.rms_eps)
        return mrsa.linear_int8(q8, s8, *m.lm_head), mrsa.add_rms_norm(delta, x, model.final_norm, cfg.rms_eps)[0]

    with torch.inference_mode():
        first = torch.where(lmk[None, :, None], m.embed[ids] + m.role, m.embed[ids])
        logits, hidden = model_by(first, lambda i, q, k, v, h: m.attend(i, q, k, v, h, pos, None))
        assert torch.equal(m(ids, pos), logits) and torch.equal(m(ids, pos, logits=False), hidden)
        # over pages: the model's own cache holds what the steps append to theirs
        dec, own = (PagedDream(m, pages=12, sequences=2, max_len=512) for _ in range(2))
        got = dec.prefill(dec.cache.seqs(0), ids)
        seqs = own.cache.seqs(0)
        own.cache.extend(seqs, 512)

        def paged(i, q, k, v, h):
            q = own.cache.append(i, seqs, k, v, q=q, inv_freq=m.inv_freq, attention_factor=m.attention_factor)
            return own.cache.attend(i, seqs, q).reshape(1, 512, -1)

        assert torch.equal(model_by(m.embed[ids], paged)[0], got)
