"""AdamW over many tensors, states in 32 or 8 bits, against the formulas in 64 bits."""

import math

import pytest
import torch

from burn_dragon_b200.train.optim import BLOCK, AdamWMany

SIZES = [1, 2, 255, 256, 257, 0, 1000, 4096, 5, 70001]


def tensors(sizes, dev, dtype, seed, scale=1.0, flat=False):
    gen = torch.Generator().manual_seed(seed)
    xs = [torch.randn(n, generator=gen) * scale for n in sizes]
    if not flat:
        return [x.to(dev, dtype) for x in xs]
    whole = torch.cat(xs).to(dev, dtype)  # views at odd places of one buffer
    return list(whole.split(sizes))


def adamw64(p, g, m, v, t, lr, b1=0.9, b2=0.999, eps=1e-8, wd=0.1):
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * wd) - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps)
    return p, m, v


def run_32(dev, pdt, gdt, flat, shadow, sizes=SIZES, steps=3):
    ps = tensors(sizes, dev, pdt, 1, 0.1, flat)
    shadows = [torch.empty_like(p, dtype=torch.bfloat16) for p in ps] if shadow else None
    opt = AdamWMany(ps, lr=1e-2, shadows=shadows)
    ref = [(p.double().cpu(), torch.zeros(p.numel(), dtype=torch.float64), torch.zeros(p.numel(), dtype=torch.float64))
           for p in ps]
    coef = torch.tensor([0.5], device=dev)
    for t in range(1, steps + 1):
        gs = tensors(sizes, dev, gdt, 10 + t, 1e-2, flat)
        gs[3] = None if t == 2 else gs[3]
        opt.step(gs, lr=1e-2 / t, grad_scale=coef if t == 3 else None)
        for i, g in enumerate(gs):
            if g is None:
                continue
            q, m, v = adamw64(*((ref[i][0],) + (g.double().cpu() * (0.5 if t == 3 else 1.0),) + ref[i][1:]), t, 1e-2 / t)
            ref[i] = (ps[i].double().cpu() if pdt == torch.bfloat16 else q, m, v)
            # one rounding of p to its type and the fp32 operations: about ten, 2^-24 each, of
            # p and of an update of at most lr * 10 / t
            size = q.abs() + 0.1 / t
            bound = (torch.finfo(pdt).eps / 2 if pdt == torch.bfloat16 else 0.0) * q.abs() + 16 * 2.0 ** -24 * size
            assert ((ps[i].double().cpu() - q).abs() <= bound).all(), (t, i)
            if shadow:
                assert torch.equal(shadows[i], ps[i].bfloat16())
            for k, want in zip(opt.moments(i), (m, v)):
                if want.numel():
                    assert ((k.double().cpu() - want).abs() <= 16 * 2.0 ** -24 * (want.abs() + want.abs().max())).all()


@pytest.mark.gpu
@pytest.mark.parametrize("pdt,gdt,flat,shadow", [(torch.float32, torch.float32, False, False),
                                                 (torch.float32, torch.bfloat16, True, True),
                                                 (torch.float32, torch.float32, True, False),
                                                 (torch.bfloat16, torch.bfloat16, False, False)])
def test_step_in_32_bits_on_the_device(pdt, gdt, flat, shadow):
    run_32("cuda", pdt, gdt, flat, shadow)


@pytest.mark.parametrize("gdt", [torch.float32, torch.bfloat16])
def test_step_in_32_bits_on_the_cpu(gdt):
    run_32("cpu", torch.float32, gdt, True, True)


@pytest.mark.gpu
def test_more_tensors_than_one_launch_names():
    run_32("cuda", torch.float32, torch.float32, True, False, sizes=[(37 * i) % 600 for i in range(1500)], steps=2)


def grid_of(opt, i):
    """The codes and scales of tensor i's moments, whole blocks."""
    lo, hi = opt.block0[i], opt.block0[i + 1]
    out = {}
    for k in ("m", "v"):
        out[k] = (opt.state[k][lo * BLOCK:hi * BLOCK].view(torch.uint8).cpu().view(-1, BLOCK),
                  opt.state[k + "_scale"][lo:hi].cpu())
    return out


def neighbours(x):
    """The e4m3 values at and around each |x| (64 bits, |x| <= 256): below and above."""
    e = torch.floor(torch.log2(x.clamp_min(2.0 ** -6)))
    unit = torch.exp2(e - 3)
    below = torch.floor(x / unit) * unit
    return below, below + unit


def run_8(dev, sizes, flat):
    ps = tensors(sizes, dev, torch.float32, 1, 0.1, flat)
    opt = AdamWMany(ps, lr=1e-2, state_bits=8, seed=7)
    for t in range(1, 4):
        gs = tensors(sizes, dev, torch.bfloat16, 20 + t, 1e-2, flat)
        before = [(p.double().cpu(),) + tuple(k.cpu() for k in opt.moments(i)) for i, p in enumerate(ps)]
        opt.step(gs)
        for i, g in enumerate(gs):
            if not g.numel():
                continue
            q = adamw64(before[i][0], g.double().cpu(), *(k.double() for k in before[i][1:]), t, 1e-2)[0]
            # what is rounded to 8 bits are the fp32 moments, each product and sum rounded by itself
            f, (m, v) = g.float().cpu(), before[i][1:]
            m, v = m * 0.9 + f * (1 - 0.9), v * 0.999 + (f * f) * (1 - 0.999)
            assert ((ps[i].double().cpu() - q).abs() <= 16 * 2.0 ** -24 * (q.abs() + 0.1)).all()
            pad = -g.numel() % BLOCK
            for k, want in (("m", m), ("v", v)):
                codes, scale = grid_of(opt, i)[k]
                want = torch.nn.functional.pad(want, (0, pad)).view(-1, BLOCK)
                amax = want.abs().amax(1)
                assert torch.equal(scale * 256, amax)
                x = torch.where(amax[:, None] > 0, want.double() / amax[:, None].double() * 256, 0.0)
                got = codes.view(torch.float8_e4m3fn).double()
                low, high = neighbours(x.abs())
                slack = 2.0 ** -19 * x.abs()
                fine = (got.abs() >= low - slack) & (got.abs() <= high + slack)
                if k == "v":
                    fine &= (x == 0) | (got >= 2.0 ** -9)
                assert fine.all() and ((got == 0) | (got.sign() == x.sign())).all()
            assert (grid_of(opt, i)["m"][0].view(-1)[g.numel():] == 0).all()  # what pads a tensor stays zero
    return opt


@pytest.mark.gpu
@pytest.mark.parametrize("flat", [False, True])
def test_step_in_8_bits_on_the_device(flat):
    run_8("cuda", SIZES, flat)


def test_step_in_8_bits_on_the_cpu():
    run_8("cpu", SIZES, False)


@pytest.mark.gpu
def test_the_device_rounds_as_the_cpu():
    """Separately rounded operations and a hash of the index: the same codes and scales, bit for bit."""
    states = []
    for dev in ("cpu", "cuda"):
        ps = tensors(SIZES, dev, torch.float32, 3, 0.1, True)
        opt = AdamWMany(ps, state_bits=8, seed=11)
        for t in range(4):
            opt.step(tensors(SIZES, dev, torch.float32, 30 + t, 1e-3))
        states.append({k: (s.view(torch.uint8) if s.dtype == torch.float8_e4m3fn else s).cpu()
                       for k, s in opt.state.items()})
    for k in states[0]:
        assert torch.equal(states[0][k], states[1][k]), k


def mean_is_kept(dev):
    """E[decode(encode(x))] = x: 4096 equal values, one per hash; five deviations of their mean."""
    n = 16 * BLOCK
    p = torch.zeros(n, device=dev)
    opt = AdamWMany([p], state_bits=8, weight_decay=0.0, betas=(0.9, 0.999))
    g = torch.full((n,), 0.37, device=dev)
    g[::BLOCK] = 1.0  # the block's largest value
    opt.step([g])
    for k, value, top in ((opt.moments(0)[0], 0.1 * 0.37, 0.1), (opt.moments(0)[1], 0.001 * 0.37 ** 2, 0.001)):
        rest = torch.ones(n, dtype=torch.bool, device=dev)
        rest[::BLOCK] = False
        x = 256 * value / top
        unit = 2.0 ** (math.floor(math.log2(x)) - 3) * top / 256
        assert abs(float(k[rest].double().mean()) - value) <= 5 * 0.5 * unit / math.sqrt(n) + 1e-6 * value


def test_rounding_keeps_the_mean_on_the_cpu():
    mean_is_kept("cpu")


@pytest.mark.gpu
def test_rounding_keeps_the_mean_on_the_device():
    mean_is_kept("cuda")


def odd_gradients(dev):
    """Zero, tiny and not finite gradients: zeros stay zeros, NaN and infinity show in their own block."""
    n = 4 * BLOCK
    p = torch.ones(n, device=dev)
    opt = AdamWMany([p], state_bits=8, weight_decay=0.0)
    g = torch.zeros(n, device=dev)
    g[BLOCK:2 * BLOCK] = 1e-30
    g[2 * BLOCK] = float("inf")
    g[3 * BLOCK] = 1e-3
    opt.step([g])
    m, v = opt.moments(0)
    assert (m[:BLOCK] == 0).all() and (v[:BLOCK] == 0).all() and (p[:BLOCK] == 1).all()
    assert m[BLOCK:2 * BLOCK].isfinite().all() and (v[BLOCK:2 * BLOCK] == 0).all()
    assert m[2 * BLOCK:3 * BLOCK].isnan().all()
    assert m[3 * BLOCK:].isfinite().all() and float(m[3 * BLOCK]) > 0 and (v[3 * BLOCK + 1:] == 0).all()


def test_odd_gradients_on_the_cpu():
    odd_gradients("cpu")


@pytest.mark.gpu
def test_odd_gradients_on_the_device():
    odd_gradients("cuda")


def fit(dev, bits):
    """A least-squares problem with badly scaled inputs."""
    gen = torch.Generator().manual_seed(0)
    x = (torch.randn(512, 64, generator=gen) * torch.logspace(-1, 1, 64)).to(dev)
    want = torch.randn(64, 8, generator=gen).to(dev)
    w = torch.zeros(64, 8, device=dev)
    opt = AdamWMany([w], lr=2e-2, weight_decay=0.0, state_bits=bits)
    for _ in range(400):
        e = x @ (w - want)
        opt.step([2 * x.t() @ e / 512])
    return float((x @ (w - want)).pow(2).mean())


def test_eight_bits_learn_like_thirty_two():
    full, eight = fit("cpu", 32), fit("cpu", 8)
    start = 2200.0
    assert full < 1e-2 * start and eight < 1e-2 * start


def test_state_round_trip_and_refusals():
    ps = [torch.zeros(300), torch.zeros(5)]
    opt = AdamWMany(ps, state_bits=8, seed=3)
    opt.step([torch.ones(300), torch.ones(5)])
    other = AdamWMany([p.clone() for p in ps], state_bits=8)
    other.load_state_dict(opt.state_dict())
    for o in (opt, other):
        o.step([torch.full((300,), 0.5), None])
    assert torch.equal(opt.params[0], other.params[0]) and other.t == 2 and other.seed == 3
    assert torch.equal(opt.state["m"].view(torch.uint8), other.state["m"].view(torch.uint8))
    with pytest.raises(ValueError, match="state 'm'"):
        AdamWMany(ps, state_bits=32).load_state_dict(opt.state_dict())
    with pytest.raises(ValueError, match="8 or 32"):
        AdamWMany(ps, state_bits=16)
    with pytest.raises(ValueError, match="at least one"):
        AdamWMany([])
    with pytest.raises(ValueError, match="contiguous fp32 or bf16"):
        AdamWMany([torch.zeros(4, 4).t()[:, :2]])
    with pytest.raises(ValueError, match="contiguous fp32 or bf16"):
        AdamWMany([torch.zeros(4, dtype=torch.float64)])
    with pytest.raises(ValueError, match="shadow"):
        AdamWMany(ps, shadows=[torch.zeros(300, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.bfloat16)])
    with pytest.raises(ValueError, match="gradients for"):
        opt.step([None])
    with pytest.raises(ValueError, match="size"):
        opt.step([torch.zeros(299), None])


@pytest.mark.gpu
def test_refusals_on_the_device():
    opt = AdamWMany([torch.zeros(300, device="cuda")])
    with pytest.raises(RuntimeError, match="gradient like its tensor"):
        opt.step([torch.zeros(299, device="cuda")])
    with pytest.raises(RuntimeError, match="fp32 or bf16"):
        opt.step([torch.zeros(300, device="cuda", dtype=torch.float64)])
    with pytest.raises(RuntimeError, match="gradient like its tensor"):
        opt.step([torch.zeros(300)])
