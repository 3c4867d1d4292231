"""AdamWMany where tensors have had different numbers of steps: each is corrected for its own, as torch.optim.AdamW does.
And the rounding of its update."""

import pytest
import torch

from burn_dragon_b200.config import DragonConfig
from burn_dragon_b200.models.adapters import AdapterBank, AdapterBDH
from burn_dragon_b200.models.bdh import BDH
from burn_dragon_b200.train.optim import AdamWMany

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
LR = 1e-2


def gradient(n, seed, dev):
    return (torch.randn(n, generator=torch.Generator().manual_seed(seed)) * 1e-2).to(dev)


def against_torch(dev, when, steps, size=300, bits=32):
    """`when(i, t)`: has tensor i a gradient at step t. Four tensors against torch.optim.AdamW in 64 bits."""
    ps = [gradient(size + i, i, dev) for i in range(4)]
    ref = [torch.nn.Parameter(p.double().cpu()) for p in ps]
    opt = AdamWMany(ps, lr=LR, weight_decay=0.1, state_bits=bits)
    want = torch.optim.AdamW(ref, lr=LR, weight_decay=0.1)
    for t in range(1, steps + 1):
        gs = [gradient(size + i, 100 * t + i, dev) if when(i, t) else None for i in range(4)]
        for q, g in zip(ref, gs):
            q.grad = None if g is None else g.double().cpu()
        want.step()
        opt.step(gs)
        own = [int(want.state[q]["step"]) if q in want.state else 0 for q in ref]
        assert opt.steps == own and opt.t == t
        for i, (p, q) in enumerate(zip(ps, ref)):
            # a step adds 16 operations of 2^-24 of p and of an update of at most 10 lr; those of m and v add up alike
            bound = own[i] * 16 * 2.0 ** -24 * (q.abs() + 10 * LR)
            assert ((p.double().cpu() - q.detach()).abs() <= bound.detach()).all(), (t, i)
    return opt


@pytest.mark.parametrize("dev", DEVICES)
def test_a_tensor_that_joins_late(dev):
    against_torch(dev, lambda i, t: i == 0 or t > 15 * i, 60)


@pytest.mark.parametrize("dev", DEVICES)
def test_tensors_that_are_stepped_rarely(dev):
    against_torch(dev, lambda i, t: t % (1, 2, 5, 7)[i] == 0, 40)


@pytest.mark.parametrize("dev", DEVICES)
def test_a_first_step_far_into_the_run(dev):
    """After 3000 steps of another tensor the first update is lr times the gradient's sign, as on step 1."""
    other, late = torch.zeros(8, device=dev), torch.zeros(300, device=dev)
    opt = AdamWMany([other, late], lr=LR, weight_decay=0.0)
    one = torch.ones(8, device=dev)
    for _ in range(3000):
        opt.step([one, None])
    g = gradient(300, 1, dev)
    opt.step([one, g])
    g = g.double()
    assert ((late.double() + LR * g / (g.abs() + 1e-8)).abs() <= 32 * 2.0 ** -24 * LR).all()
    assert opt.steps == [3001, 1]


@pytest.mark.parametrize("dev", DEVICES)
def test_eight_bits_correct_each_tensors_own_steps_too(dev):
    ps = [torch.zeros(512, device=dev), torch.zeros(512, device=dev)]
    opt = AdamWMany(ps, lr=LR, weight_decay=0.0, state_bits=8)
    g = [gradient(512, 5, dev), gradient(512, 6, dev)]
    for _ in range(50):
        opt.step([g[0], None])
    opt.step(g)
    want = -LR * g[1].double() / (g[1].double().abs() + 1e-8)
    assert ((ps[1].double() - want).abs() <= 32 * 2.0 ** -24 * LR).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("pdt,gdt,shadow", [(torch.float32, torch.float32, False), (torch.float32, torch.bfloat16, True),
                                            (torch.bfloat16, torch.bfloat16, False)])
def test_types_and_odd_sizes_with_steps_of_their_own(dev, pdt, gdt, shadow):
    sizes = [1, 2, 255, 256, 257, 0, 1000, 4096, 5, 70001]
    flat = (torch.randn(sum(sizes), generator=torch.Generator().manual_seed(1)) * 0.1).to(dev, pdt)
    ps = list(flat.split(sizes))  # views at odd places of one buffer
    shadows = [torch.empty_like(p, dtype=torch.bfloat16) for p in ps] if shadow else None
    opt = AdamWMany(ps, lr=LR, shadows=shadows)
    own = [0] * len(sizes)
    ref = [(p.double().cpu(), torch.zeros(p.numel(), dtype=torch.float64), torch.zeros(p.numel(), dtype=torch.float64))
           for p in ps]
    coef = torch.tensor([0.5], device=dev)
    for t in range(1, 5):
        gs = [None if (i + t) % 3 == 0 else gradient(n, 10 * t + i, dev).to(gdt) for i, n in enumerate(sizes)]
        opt.step(gs, lr=LR / t, grad_scale=coef if t == 3 else None)
        for i, g in enumerate(gs):
            if g is None:
                continue
            own[i] += 1
            p, m, v = ref[i]
            g = g.double().cpu() * (0.5 if t == 3 else 1.0)
            m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
            q = p * (1 - LR / t * 0.1) - LR / t * (m / (1 - 0.9 ** own[i])) / ((v / (1 - 0.999 ** own[i])).sqrt() + 1e-8)
            # one rounding of p to its type and about ten fp32 operations on p and on an update of at most 10 lr
            bound = (torch.finfo(pdt).eps / 2 if pdt == torch.bfloat16 else 0.0) * q.abs() + 16 * 2.0 ** -24 * (q.abs() + 0.1 / t)
            assert ((ps[i].double().cpu() - q).abs() <= bound).all(), (t, i)
            if shadow:
                assert torch.equal(shadows[i], ps[i].bfloat16())
            ref[i] = (ps[i].double().cpu(), m, v)
    assert opt.steps == own


def test_step_counts_are_saved_and_loaded():
    ps = [torch.zeros(300), torch.zeros(5)]
    opt = AdamWMany(ps, state_bits=8)
    opt.step([torch.ones(300), None])
    opt.step([torch.ones(300), torch.ones(5)])
    other = AdamWMany([p.clone() for p in ps], state_bits=8)
    other.load_state_dict(opt.state_dict())
    assert other.steps == [2, 1] and other.t == 2
    for o in (opt, other):
        o.step([torch.ones(300), torch.ones(5)])
    assert torch.equal(opt.params[1], other.params[1])
    old = {k: v for k, v in opt.state_dict().items() if k != "steps"}  # saved before the counts were kept
    other.load_state_dict(old)
    assert other.steps == [3, 3]
    with pytest.raises(ValueError, match="step counts"):
        other.load_state_dict({**opt.state_dict(), "steps": [1]})
    m = other.state["m"].clone()
    with pytest.raises(ValueError, match="v_scale"):  # nothing is taken over from a state that does not fit
        other.load_state_dict({**opt.state_dict(), "m": torch.zeros_like(m), "v_scale": torch.zeros(9)})
    assert torch.equal(other.state["m"].view(torch.uint8), m.view(torch.uint8))


def test_an_adapter_trains_as_it_would_alone():
    """A bank's adapter that joins after 30 steps of another one takes the steps of a fresh bank."""
    cfg = DragonConfig(n_layer=2, n_embd=32, n_head=2, mlp_internal_dim_multiplier=8, dropout=0.0)
    model = BDH(cfg, seed=1)
    x = torch.randint(0, 256, (1, 17), generator=torch.Generator().manual_seed(4))
    moved = []
    for before in (0, 30):
        net = AdapterBDH(model, AdapterBank(cfg, 2, rank=4, seed=3))
        opt = net.optimizer(lr=1e-2)
        for _ in range(before):
            net.train_step(opt, x[:, :-1], x[:, 1:], [0])
        for _ in range(5):
            net.train_step(opt, x[:, :-1], x[:, 1:], [1])
        moved.append({n: t[1].clone() for n, t in net.bank.master.items()})
    for n in moved[0]:
        assert torch.equal(moved[0][n], moved[1][n])


@pytest.mark.gpu
def test_a_step_in_32_bits_rounds_root_and_quotient_correctly():
    """From p = 0 the step is -(m lr / bc1) / (sqrt(v / bc2) + eps), operation by operation in fp32."""
    p, g = torch.zeros(70001, device="cuda"), gradient(70001, 3, "cuda")
    opt = AdamWMany([p], lr=LR, weight_decay=0.1)
    opt.step([g])
    m, v = opt.moments(0)
    f32 = lambda x: torch.tensor(x, dtype=torch.float32, device="cuda")  # noqa: E731
    want = (m * f32(LR / (1 - 0.9))) / ((v * f32(1 / (1 - 0.999))).sqrt() + f32(1e-8))
    assert torch.equal(p, -want)
