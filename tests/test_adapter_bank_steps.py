"""AdapterBDH: what a training step and a generation do at their edges."""

import pytest
import torch

from burn_dragon_b200.config import DragonConfig
from burn_dragon_b200.models import reference as R
from burn_dragon_b200.models.adapters import AdapterBank, AdapterBDH
from burn_dragon_b200.models.bdh import BDH


def make(G=3, **kw):
    cfg = DragonConfig(**{**dict(n_layer=2, n_embd=32, n_head=2, mlp_internal_dim_multiplier=8, dropout=0.0), **kw})
    model = BDH(cfg, seed=1)
    return model, AdapterBDH(model, AdapterBank(cfg, G, rank=4))


TOKENS = torch.randint(0, 256, (2, 9), generator=torch.Generator().manual_seed(4))


def test_a_plan_of_other_adapters_is_refused():
    _, net = make()
    opt = net.optimizer()
    x, y = TOKENS[:, :-1], TOKENS[:, 1:]
    net.train_step(opt, x, y, range(2), batch=net.batch([0, 1], 8))
    before = {n: t.clone() for n, t in net.bank.master.items()}
    for plan in (net.batch([0, 2], 8), net.batch([1, 0], 8), net.batch([0, 1], 9)):
        with pytest.raises(ValueError, match="planned for other"):
            net.train_step(opt, x, y, [0, 1], batch=plan)
    assert all(torch.equal(t, before[n]) for n, t in net.bank.master.items()) and opt.t == 1
    net.train_step(opt, x, y, [0, 1], batch=net.batch([0, 0, 1, 1], 4))  # the same adapter for every row


def test_a_step_trains_with_the_models_dropout():
    """At a rate of 1 the layers add nothing, which needs no equal random numbers: the loss is the model's own."""
    for mode, rate in ((True, 1.0), (False, 0.0)):
        model, net = make(dropout=1.0)
        model.train(mode)
        x, y = TOKENS[:, :-1], TOKENS[:, 1:]
        want = float(model.loss(x, y).detach())
        assert abs(float(net.train_step(net.optimizer(), x, y, [0, 1])) - want) < 1e-5
        p = {k: v.detach() for k, v in model.param_dict().items() if v is not None}
        model.cfg.dropout = rate
        assert abs(float(R.cross_entropy(R.bdh_forward(x, p, model.cfg, training=True)[0], y)) - want) < 1e-5
    model, net = make(dropout=0.5)
    losses = {float(net.train_step(net.optimizer(lr=0.0), TOKENS[:, :-1], TOKENS[:, 1:], [0, 1])) for _ in range(4)}
    assert len(losses) == 4  # drawn anew each step
    logits = [net.forward(TOKENS, net.batch([0, 1], 9)) for _ in range(2)]
    assert torch.equal(*logits)  # and not in answers


@pytest.mark.parametrize("prompts", [[[1, 2], [3, 4]], [[1, 2, 3], [4]]])
def test_no_new_tokens_are_an_empty_answer(prompts):
    _, net = make()
    assert net.generate(prompts, [0, -1], 0) == ([[], []], [[], []])
    out, lp = net.generate(prompts, [0, -1], 1)
    assert [len(o) for o in out] == [1, 1] == [len(v) for v in lp]
