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
    for plan in (net.batch([0, 2], 8), net.batch([1, 0], 8), net.batch([0, 1], 9), net.batch([0, 0, 1, 1], 4)):
        with pytest.raises(ValueError, match="planned for other"):
            net.train_step(opt, x, y, [0, 1], batch=plan)
    assert all(torch.equal(t, before[n]) for n, t in net.bank.master.items()) and opt.t == 1
