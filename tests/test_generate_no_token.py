"""Generation where a row's logits leave nothing to draw from: sample_tokens answers -1, which is no token id."""

import pytest
import torch

from burn_dragon_b200.config import DragonConfig
from burn_dragon_b200.models.adapters import AdapterBank, AdapterBDH
from burn_dragon_b200.models.bdh import BDH
from burn_dragon_b200.models.generate import Generator


def small(dev="cpu"):
    cfg = DragonConfig(n_layer=2, n_embd=64, n_head=2, mlp_internal_dim_multiplier=8, dropout=0.0, rotary_embedding="rope")
    return BDH(cfg, device=dev, seed=1)


class Breaking(Generator):
    """A generator whose first row has NaN logits in its third decode step only."""

    def __init__(self, model, broken=0):
        super().__init__(model)
        self.steps, self.read, self.broken = 0, [], broken

    def decode_step(self, tokens, state):
        assert int(tokens.min()) >= 0 and int(tokens.max()) < self.cfg.vocab_size  # what the model reads is a token
        self.read.append(tokens.tolist())
        logits = super().decode_step(tokens, state).clone()
        self.steps += 1
        if self.steps == 3:
            logits[self.broken] = float("nan")
        return logits


@pytest.mark.parametrize("top_p,min_p", [(0.9, None), (None, 0.05)])
def test_a_row_without_a_token_ends_and_the_others_go_on(top_p, min_p):
    x = torch.tensor([[1, 2, 3], [4, 5, 6]])
    whole = Generator(small()).generate(x, 8, temperature=0.8, top_p=top_p, min_p=min_p, seed=3)
    out = Breaking(small()).generate(x, 8, temperature=0.8, top_p=top_p, min_p=min_p, seed=3, device_buffer_tokens=3)
    assert torch.equal(out[1], whole[1])
    assert torch.equal(out[0, :3], whole[0, :3]) and out[0, 3:].tolist() == [-1] * 5


def test_a_stream_without_a_token_raises_after_what_it_has():
    seen = []
    whole = Generator(small()).generate_stream([1, 2, 3], 8, temperature=0.8, top_p=0.9, seed=3)
    with pytest.raises(RuntimeError, match="no token to draw"):
        Breaking(small()).generate_stream([1, 2, 3], 8, chunk_tokens=2, temperature=0.8, top_p=0.9, seed=3,
                                          on_chunk=seen.extend)
    assert seen == whole[3:6]
    # a stop token before it ends the answer as always
    stop = whole[4]
    got = Breaking(small()).generate_stream([1, 2, 3], 8, chunk_tokens=4, temperature=0.8, top_p=0.9, seed=3, stop_token=stop)
    assert got == whole[:whole.index(stop, 3) + 1]


def test_a_request_of_a_bank_without_a_token_ends(monkeypatch):
    model = small()
    prompts, ids = [[1, 2, 3], [7, 8], [9]], [0, -1, 1]
    whole, lp_whole = AdapterBDH(model, AdapterBank(model.cfg, 2, rank=4)).generate(prompts, ids, 5, temperature=0.9, seed=2)
    net = AdapterBDH(model, AdapterBank(model.cfg, 2, rank=4))
    plain, calls = net.forward, []

    def forward(tokens, batch, state=None, work=None):
        assert int(tokens.min()) >= 0
        logits = plain(tokens, batch, state, work).clone()
        calls.append(1)
        if len(calls) == 4:
            logits[1] = float("nan")
        return logits

    monkeypatch.setattr(net, "forward", forward)
    out, lp = net.generate(prompts, ids, 5, temperature=0.9, seed=2)
    assert out[0] == whole[0] and out[2] == whole[2] and lp[0] == lp_whole[0] and lp[2] == lp_whole[2]
    assert out[1][:2] == whole[1][:2] and out[1][2:] == [-1] * 3 and lp[1][2:] == [float("-inf")] * 3


@pytest.mark.gpu
def test_a_row_without_a_token_on_the_device():
    x = torch.tensor([[1, 2, 3], [4, 5, 6]], device="cuda")
    whole = Generator(small("cuda")).generate(x, 8, temperature=0.8, top_p=0.9, seed=3)
    g = Breaking(small("cuda"))
    assert g._fused_ok
    g.steps = -3  # the prompt is read in decode steps too
    out = g.generate(x, 8, temperature=0.8, top_p=0.9, seed=3)
    assert torch.equal(out[1], whole[1]) and out[0, 3:].tolist() == [-1] * 5
