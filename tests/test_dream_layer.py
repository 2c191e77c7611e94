"""What a layer of the Dream-shaped model is made of, on the CPU: the steps that a subclass may put others in place of."""

import torch


def test_layer_takes_the_attention_of_a_subclass(mrsa):
    from mrsa_b200.dream_forward import DreamConfig, DreamForward

    class Own(DreamForward):
        def __init__(self):
            self.cfg, self.layers = DreamConfig(), [{"in_norm": torch.tensor(2.0)}]

        def rms_norm(self, x, weight):
            return x * weight

        def attention(self, idx, h, position_ids, key_valid):
            return h + position_ids if key_valid is None else h

        def leave(self, idx, o, x):
            return o, x

    m, x, pos = Own(), torch.ones(1, 3, 4), torch.arange(3.0)[None, :, None]
    o, kept = m.layer(0, x, pos, None)
    assert kept is x and torch.equal(o, 2 * x + pos)
    assert torch.equal(m.layer(0, x, pos, pos > 0)[0], 2 * x)
