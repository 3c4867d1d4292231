"""A bank of adapters on one frozen model: against the model with the adapter folded in, training and serving."""

import pytest
import torch

from burn_dragon_b200.config import DragonConfig
from burn_dragon_b200.models.adapters import AdapterBank, AdapterBDH
from burn_dragon_b200.models.bdh import BDH
from burn_dragon_b200.models.generate import Generator


def small():
    cfg = DragonConfig.tiny()
    cfg.n_embd, cfg.n_head, cfg.n_layer = 32, 2, 2
    cfg.mlp_internal_dim_multiplier = 8  # 256 latents
    return cfg


def make(dev="cpu", G=3, seed=0):
    model = BDH(small(), device=dev, seed=1)
    bank = AdapterBank(model.cfg, G, rank=4, device=dev, seed=seed)
    gen = torch.Generator().manual_seed(9)
    for name, t in bank.master.items():
        if name.endswith(".b"):
            t.copy_(torch.randn(t.shape, generator=gen) * 0.02)
            if bank.work[name] is not t:
                bank.work[name].copy_(t)
    return model, bank


def folded(model, bank, g):
    """The same model with adapter g added to its projections."""
    p = {k: v if v is None else v.detach().clone() for k, v in model.param_dict().items()}
    for n in ("encoder", "encoder_v", "decoder"):
        a, b = bank.master[n + ".a"][g], bank.master[n + ".b"][g]
        p[n] += bank.scale * a.transpose(-1, -2) @ b
    return p


def test_sequences_answer_as_with_their_adapter_folded_in():
    from burn_dragon_b200.models import reference as R

    model, bank = make()
    net = AdapterBDH(model, bank)
    tokens = torch.randint(0, 256, (4, 12), generator=torch.Generator().manual_seed(2))
    ids = [2, -1, 0, 2]
    got = net.forward(tokens, net.batch(ids, 12))
    for i, g in enumerate(ids):
        p = folded(model, bank, g) if g >= 0 else model.param_dict()
        want = R.bdh_forward(tokens[i:i + 1], p, model.cfg)[0]
        assert torch.allclose(got[i:i + 1], want, atol=1e-4, rtol=1e-4)


def test_single_tokens_continue_the_prompt():
    from burn_dragon_b200.models.state import ModelState

    model, bank = make()
    net = AdapterBDH(model, bank)
    tokens = torch.randint(0, 256, (3, 9), generator=torch.Generator().manual_seed(3))
    ids = [1, 0, -1]
    want = net.forward(tokens, net.batch(ids, 9))
    state = ModelState.empty()
    parts = [net.forward(tokens[:, :5], net.batch(ids, 5), state)]
    one = net.batch(ids, 1)
    parts += [net.forward(tokens[:, t:t + 1], one, state) for t in range(5, 9)]
    assert torch.allclose(torch.cat(parts, 1), want, atol=1e-4, rtol=1e-4)


def test_training_moves_only_the_adapters_of_the_batch():
    model, bank = make(G=3)
    net = AdapterBDH(model, bank)
    before = {n: t.clone() for n, t in bank.master.items()}
    frozen = {n: t.clone() for n, t in net.weights.items()}
    opt = net.optimizer(lr=1e-2, state_bits=8)
    x = torch.randint(0, 256, (2, 17), generator=torch.Generator().manual_seed(4))
    losses = [float(net.train_step(opt, x[:, :-1], x[:, 1:], [0, 2])) for _ in range(12)]
    assert losses[-1] < losses[0]
    for n, t in bank.master.items():
        assert torch.equal(t[1], before[n][1]) and not torch.equal(t[0], before[n][0])
    assert all(torch.equal(net.weights[n], frozen[n]) for n in frozen)


def test_serving_requests_of_different_lengths_and_settings():
    model, bank = make()
    net = AdapterBDH(model, bank)
    prompts, ids = [[1, 2, 3, 4, 5], [7], [9, 8, 7]], [0, -1, 2]
    out, lp = net.generate(prompts, ids, 6, temperature=[0.0, 1.0, 0.7], top_k=[0, 5, 0], top_p=[1.0, 0.9, 0.5], seed=5)
    assert [len(o) for o in out] == [6, 6, 6] and lp[0] == [0.0] * 6 and all(v <= 0 for v in lp[1] + lp[2])
    again, _ = net.generate(prompts, ids, 6, temperature=[0.0, 1.0, 0.7], top_k=[0, 5, 0], top_p=[1.0, 0.9, 0.5], seed=5)
    assert out == again
    alone, _ = net.generate(prompts[:1], ids[:1], 6, temperature=0.0)
    assert alone[0] == out[0]  # greedy: as by itself
    with pytest.raises(ValueError, match="empty prompts"):
        net.generate([[1], []], [0, 0], 2)


def test_scaffold_adapters_load():
    model, bank = make()
    src = {n: torch.randn(*(t.shape[1:-2] + ((t.shape[-1], t.shape[-2]) if n.endswith(".a") else t.shape[-2:])))
           for n, t in bank.master.items()}
    bank.load_scaffold(1, src)
    for n, t in bank.master.items():
        assert torch.equal(t[1], src[n].transpose(-1, -2) if n.endswith(".a") else src[n])


def test_unsupported_models_are_refused():
    cfg = small()
    cfg.mhc_streams = 2
    model = BDH(small(), seed=1)
    model.cfg = cfg
    with pytest.raises(ValueError, match="mHC"):
        AdapterBDH(model, AdapterBank(cfg, 1))
    with pytest.raises(ValueError, match="scaling"):
        AdapterBank(cfg, 1, scaling="other")


def test_generator_with_top_p_and_min_p():
    model = BDH(small(), seed=1)
    g = Generator(model)
    x = torch.tensor([[1, 2, 3], [4, 5, 6]])
    out = g.generate(x, 5, temperature=0.8, top_p=0.9, seed=3)
    assert out.shape == (2, 5) and torch.equal(out, g.generate(x, 5, temperature=0.8, top_p=0.9, seed=3))
    greedy = g.generate(x, 5)
    assert torch.equal(g.generate(x, 5, temperature=0.8, top_p=0.0, seed=3), greedy)  # one token is left
    assert torch.equal(g.generate(x, 5, temperature=0.8, min_p=1.0, seed=3), greedy)


def test_cli_trains_and_serves(capsys):
    from burn_dragon_b200.cli.adapters import main

    main(["--text", "abcabc", "--text", "0123", "--steps", "3", "--length", "8", "--max-tokens", "4", "--rank", "2",
          "--state-bits", "8", "--temperature", "0.7", "--top-p", "0.9"])
    text = capsys.readouterr().out
    assert "step 2: loss" in text and "adapter 0:" in text and "adapter 1:" in text


@pytest.mark.gpu
def test_device_path_follows_the_cpu_path():
    """bf16 projections against fp32 ones: each of the 6 rounds inputs and outputs to 2^-8; logits are of size one."""
    model, bank = make()
    gpu_model, gpu_bank = make("cuda")
    tokens = torch.randint(0, 256, (4, 40), generator=torch.Generator().manual_seed(2))
    ids = [2, -1, 0, 1]
    want = AdapterBDH(model, bank)
    got = AdapterBDH(gpu_model, gpu_bank)
    a = want.forward(tokens, want.batch(ids, 40))
    b = got.forward(tokens.cuda(), got.batch(ids, 40)).cpu()
    assert (a - b).abs().max() <= 6 * 4 * 2.0 ** -8 * a.abs().max()
    opt = got.optimizer(lr=1e-2, state_bits=8)
    x = tokens[:2].cuda()
    losses = [float(got.train_step(opt, x[:, :-1], x[:, 1:], [0, 2])) for _ in range(12)]
    assert losses[-1] < losses[0]
    out, lp = got.generate([[1, 2, 3], [4]], [0, -1], 5, temperature=0.9, top_p=0.9)
    assert [len(o) for o in out] == [5, 5]
