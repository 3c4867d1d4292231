"""Adapters taken over from random-scaffold models answer as those models do."""

import copy

import pytest
import torch

from burn_dragon_b200.config import DragonConfig, RandomScaffoldConfig
from burn_dragon_b200.models.adapters import AdapterBank, AdapterBDH
from burn_dragon_b200.models.bdh import BDH, record_name


def scaffold_model(seed, scaling="standard", trainable_gain=True, dev="cpu", scaffold_seed=20260729):
    rs = RandomScaffoldConfig(enabled=True, seed=scaffold_seed, rank=4, alpha=16.0, scaling=scaling,
                              trainable_gain=trainable_gain)
    cfg = DragonConfig(n_layer=2, n_embd=32, n_head=2, mlp_internal_dim_multiplier=8, dropout=0.0,
                       rotary_embedding="rope", init_std=0.1, random_scaffold=rs)
    model = BDH(cfg, device=dev, seed=1)  # one seed: the same embedding, head and norms
    gen = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for n in ("encoder", "encoder_v", "decoder"):
            b = getattr(model, n + "_b")
            b.copy_(torch.randn(b.shape, generator=gen) * 0.05)
            if trainable_gain:
                getattr(model, n + "_gain").fill_(1.0 + 0.3 * seed)
    model.store.refresh_shadow()
    return model


def close(got, want):
    assert (got - want).abs().max() <= 1e-5 * want.abs().max() + 1e-6


TOKENS = torch.randint(0, 256, (3, 11), generator=torch.Generator().manual_seed(2))


@pytest.mark.parametrize("own", ["standard", "rank_stabilized"])
@pytest.mark.parametrize("scaling", ["standard", "rank_stabilized"])
@pytest.mark.parametrize("trainable_gain", [True, False])
@pytest.mark.parametrize("base", ["itself", "another of the seed", "a dense model of W_seed"])
def test_two_scaffold_models_in_one_batch(base, trainable_gain, scaling, own):
    models = [scaffold_model(1, scaling, trainable_gain), scaffold_model(2, scaling, trainable_gain)]
    fresh = scaffold_model(0, scaling, trainable_gain)
    with torch.no_grad():
        for n in ("encoder", "encoder_v", "decoder"):
            getattr(fresh, n + "_b").zero_()
    host = {"itself": models[0], "another of the seed": fresh,
            "a dense model of W_seed": fresh.fold_scaffold_for_inference()}[base]
    bank = AdapterBank(models[0].cfg, 2, rank=4, scaling=own)  # the bank's own scaling is not the scaffold's
    for g, m in enumerate(models):
        bank.load_scaffold(g, m)
    net = AdapterBDH(host, bank)
    got = net.forward(TOKENS, net.batch([1, -1, 0], 11))
    close(got[0:1], models[1](TOKENS[0:1]).detach())
    close(got[1:2], fresh(TOKENS[1:2]).detach())
    close(got[2:3], models[0](TOKENS[2:3]).detach())


def test_by_the_names_of_the_state_dict_and_of_the_record():
    model = scaffold_model(1)
    want = model(TOKENS).detach()
    for tensors in (model.state_dict(), {record_name(k): v for k, v in model.state_dict().items()}):
        bank = AdapterBank(model.cfg, 1, rank=4)
        bank.load_scaffold(0, tensors)
        net = AdapterBDH(model, bank)
        close(net.forward(TOKENS, net.batch([0, 0, 0], 11)), want)
    dense = copy.deepcopy(model.cfg)
    dense.random_scaffold.enabled = False  # a configuration that does not know the scaffold: its scaling is given
    bank = AdapterBank(dense, 1, rank=4)
    bank.load_scaffold(0, model.state_dict(), scale=model.cfg.random_scaffold.adapter_scale())
    net = AdapterBDH(model, bank)
    close(net.forward(TOKENS, net.batch([0, 0, 0], 11)), want)


def test_adapters_loaded_after_the_model_was_wrapped():
    model = scaffold_model(1)
    bank = AdapterBank(model.cfg, 2, rank=4)
    net = AdapterBDH(model, bank)
    close(net.forward(TOKENS, net.batch([0, -1, 1], 11)), model(TOKENS).detach())  # fresh adapters beside the whole model
    bank.load_scaffold(1, scaffold_model(2))
    close(net.forward(TOKENS, net.batch([1, 1, 1], 11)), scaffold_model(2)(TOKENS).detach())


def test_training_goes_on_from_a_scaffolds_adapter():
    model = scaffold_model(1)
    bank = AdapterBank(model.cfg, 2, rank=4)
    bank.load_scaffold(0, model)
    net = AdapterBDH(model, bank)
    opt = net.optimizer(lr=1e-2)
    x = torch.randint(0, 256, (1, 17), generator=torch.Generator().manual_seed(4))
    first = float(model.loss(x[:, :-1], x[:, 1:]).detach())
    losses = [float(net.train_step(opt, x[:, :-1], x[:, 1:], [0])) for _ in range(8)]
    assert abs(losses[0] - first) < 1e-4 and losses[-1] < losses[0]


def test_what_does_not_belong_together_is_refused():
    model = scaffold_model(1)
    bank = AdapterBank(model.cfg, 2, rank=4)
    bank.load_scaffold(0, model)
    with pytest.raises(ValueError, match="share W_seed"):
        bank.load_scaffold(1, scaffold_model(1, scaffold_seed=7))
    with pytest.raises(ValueError, match="not the W_seed"):
        AdapterBDH(scaffold_model(1, scaffold_seed=7), bank)
    with pytest.raises(ValueError, match="not the W_seed"):
        AdapterBDH(model.fold_scaffold_for_inference(), bank)  # its own adapter is folded in
    with pytest.raises(ValueError, match="bank's adapters are"):
        AdapterBank(model.cfg, 1, rank=8).load_scaffold(0, model)
    with pytest.raises(ValueError, match="random-scaffold model"):
        bank.load_scaffold(0, model.fold_scaffold_for_inference())
    with pytest.raises(KeyError, match="encoder.a"):
        bank.load_scaffold(0, {})
    with torch.no_grad():
        model.decoder_gain.zero_()
    with pytest.raises(ValueError, match="gain of 0.0"):
        bank.load_scaffold(1, model)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("from_scaffold", [True, False])
def test_a_bank_is_saved_and_loaded(from_scaffold, dev, tmp_path):
    model = scaffold_model(1, dev=dev)
    bank = AdapterBank(model.cfg, 2, rank=4, alpha=3.0, device=dev, seed=8)
    if from_scaffold:
        bank.load_scaffold(0, model)
    net = AdapterBDH(model, bank)
    opt = net.optimizer(lr=1e-2)
    tokens = TOKENS.to(dev)
    for _ in range(3):
        net.train_step(opt, tokens[:, :-1], tokens[:, 1:], [0, 1, -1])
    want = net.forward(tokens, net.batch([0, 1, -1], 11))
    torch.save(bank.state_dict(), tmp_path / "bank.pt")
    other = AdapterBank(model.cfg, 2, rank=4, device=dev)
    before = AdapterBDH(model, other)
    other.load_state_dict(torch.load(tmp_path / "bank.pt"))
    for got in (before, AdapterBDH(model, other)):
        assert torch.equal(got.forward(tokens, got.batch([0, 1, -1], 11)), want)
    with pytest.raises(ValueError, match="the bank's is"):
        AdapterBank(model.cfg, 3, rank=4, device=dev).load_state_dict(bank.state_dict())


@pytest.mark.gpu
def test_on_the_device():
    """bf16 projections against the fp32 model: each of the 6 rounds inputs, weights and outputs to 2^-8."""
    models = [scaffold_model(1, dev="cuda"), scaffold_model(2, dev="cuda")]
    bank = AdapterBank(models[0].cfg, 2, rank=4, device="cuda")
    for g, m in enumerate(models):
        bank.load_scaffold(g, m)
    net = AdapterBDH(models[0], bank)
    got = net.forward(TOKENS.cuda(), net.batch([1, 0, 0], 11)).cpu()
    for i, m in enumerate((models[1], models[0], models[0])):
        want = m(TOKENS[i:i + 1].cuda()).detach().cpu()
        assert (got[i:i + 1] - want).abs().max() <= 6 * 4 * 2.0 ** -8 * want.abs().max()
