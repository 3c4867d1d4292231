"""linear_act, gated_linear and 8-bit activations as a user's program meets them: refusals, layouts, streams, graphs, parts
of the gradients, numbers that are not finite; and in the models that call them."""

import pytest
import torch
import torch.nn.functional as F

from burn_dragon_b200.config import DragonConfig, TrainingConfig
from burn_dragon_b200.models.dragon_runtime import DragonRuntime, RuntimeState
from burn_dragon_b200.models.micro_transformer import MicroTransformerBlock
from burn_dragon_b200.ops.act8 import activations_in_8bit
from burn_dragon_b200.ops.feed_forward import gated_linear, linear_act
from burn_dragon_b200.train.runtime_trainer import RuntimeTrainer

BF = torch.bfloat16


def rn(*shape, seed=0, dev="cpu", dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape))).to(dtype).to(dev)


def refusals(dev, dtype):
    x, w, b = rn(5, 16, dev=dev, dtype=dtype), rn(16, 24, dev=dev, dtype=dtype), rn(24, dev=dev, dtype=dtype)
    heads = rn(3, 16, 24, dev=dev, dtype=dtype)
    for call in (lambda: linear_act(x, w.t()), lambda: linear_act(x, w, b[:-1]), lambda: linear_act(x, w, "b"),
                 lambda: linear_act(x, w, activation="tanh"), lambda: linear_act(x, w, keep="4bit"),
                 lambda: linear_act(x, w, residual=x), lambda: linear_act(x, heads),
                 lambda: gated_linear(x, w, w[:, :8]), lambda: gated_linear(x, w, w, z=x[:3]),
                 lambda: gated_linear(x, w, w, up_activation="silu"), lambda: gated_linear(x, heads, heads, z=rn(5, 2, 16, dev=dev, dtype=dtype)),
                 lambda: gated_linear(x, heads, heads, b), lambda: gated_linear(x, heads, w)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        linear_act(x, w.double())
    with pytest.raises(TypeError):
        gated_linear(x, w, w, z=x.double())


def test_refusals_on_the_cpu():
    refusals("cpu", torch.float32)


@pytest.mark.gpu
def test_refusals_on_the_device():
    refusals("cuda", BF)
    x, w = rn(5, 16, dev="cuda"), rn(16, 24, dev="cuda")
    with pytest.raises(TypeError):
        linear_act(x, w)  # fp32
    x, w = x.to(BF), w.to(BF)
    with pytest.raises(ValueError):
        linear_act(x, w.cpu())
    with pytest.raises(TypeError):
        linear_act(x, w, rn(24, dev="cuda").double())
    import torch.autograd.forward_ad as fad

    with fad.dual_level(), pytest.raises(NotImplementedError):
        linear_act(fad.make_dual(x, torch.ones_like(x)), w)
    x.requires_grad_()
    (g,) = torch.autograd.grad(linear_act(x, w, activation="silu").float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()


@pytest.mark.gpu
def test_layouts_that_are_read_as_they_lie_or_copied():
    M, K, N = 37, 64, 72
    x, w, b, r = rn(M, K, dev="cuda", dtype=BF), rn(K, N, dev="cuda", dtype=BF), rn(N, dev="cuda", dtype=BF), rn(M, N, dev="cuda", dtype=BF)
    want = linear_act(x, w, b, "gelu", residual=r)
    odd = lambda t: torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)  # noqa: E731
    wide = torch.zeros(M, K + 8, dtype=BF, device="cuda")
    wide[:, :K] = x
    for xs in (wide[:, :K], odd(x), x.t().contiguous().t()):
        assert torch.equal(linear_act(xs, w, b, "gelu", residual=r), want)
    big = torch.zeros(K, N + 24, dtype=BF, device="cuda")
    big[:, 8:8 + N] = w
    for ws in (big[:, 8:8 + N], odd(w), w.t().contiguous().t(), odd(w.t().contiguous()).t()):
        assert torch.equal(linear_act(x, ws, b, "gelu", residual=r), want)
    assert torch.equal(linear_act(x, w, odd(b), "gelu", residual=odd(r)), want)
    assert torch.equal(linear_act(x.view(1, M, K), w, b, "gelu", residual=r.view(1, M, N))[0], want)
    assert torch.equal(linear_act(x[3], w, b, "gelu", residual=r[3]), linear_act(x[3:4], w, b, "gelu", residual=r[3:4])[0])
    # rows behind the batch's, and columns beside a padded one's, are left alone: outputs are whole tensors of their own
    assert linear_act(x[:0], w).shape == (0, N) and gated_linear(x[:0], w, w).shape == (0, N)
    for rows in (x[:0], x):
        rows = rows.detach().requires_grad_()
        w2 = w.detach().requires_grad_()
        gx, gw = torch.autograd.grad(linear_act(rows, w2, activation="silu").float().sum(), (rows, w2))
        assert gx.shape == rows.shape and gw.shape == w.shape and (rows.numel() or not gw.any())


@pytest.mark.gpu
@pytest.mark.parametrize("keep", ["recompute", "16bit", "8bit"])
def test_parts_of_the_gradients(keep):
    x, z = rn(140, 3, 64, dev="cuda", dtype=BF), rn(140, 64, seed=1, dev="cuda", dtype=BF)
    wg, wu = rn(3, 64, 96, seed=2, dev="cuda", dtype=BF) / 8, rn(3, 64, 96, seed=3, dev="cuda", dtype=BF) / 8
    bg, bu = rn(3, 96, seed=4, dev="cuda"), rn(3, 96, seed=5, dev="cuda")
    dy = rn(140, 3, 96, seed=6, dev="cuda", dtype=BF)
    leaves = [x, z, wg, wu, bg, bu]
    call = lambda: gated_linear(x, wg, wu, bg, bu, z=z, activation="silu", keep=keep)  # noqa: E731
    for t in leaves:
        t.requires_grad_()
    whole = torch.autograd.grad(call(), leaves, dy)
    again = torch.autograd.grad(call(), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(whole, again))  # no atomics: every bit the same
    for i, t in enumerate(leaves):
        for o in leaves:
            o.requires_grad_(o is t)
        (one,) = torch.autograd.grad(call(), t, dy)
        torch.testing.assert_close(one, whole[i], rtol=2.0 ** -7, atol=1e-6)  # one product may be split otherwise than two
    for o in leaves:
        o.requires_grad_()
    summed = torch.autograd.grad(call().float().sum(), leaves)  # an expanded gradient
    ones = torch.autograd.grad(call(), leaves, torch.ones_like(dy))
    assert all(torch.equal(a, b) for a, b in zip(summed, ones))


@pytest.mark.gpu
def test_numbers_that_are_not_finite_stay_in_their_rows():
    for M in (7, 200):
        x, w = rn(M, 64, dev="cuda", dtype=BF), rn(64, 136, dev="cuda", dtype=BF)
        fine = {a: linear_act(x, w, None, a) for a in ("none", "relu", "silu", "gelu")}
        bad = x.clone()
        bad[3, 5], bad[4, 0] = float("nan"), float("inf")
        for a, want in fine.items():
            got = linear_act(bad, w, None, a)
            keep = [i for i in range(M) if i not in (3, 4)]
            assert torch.equal(got[keep], want[keep])
            assert got[3].isnan().all() and not got[4].isfinite().all()
        got = gated_linear(bad, w, w, activation="relu", up_activation="relu")
        assert got[3].isnan().all() and got[keep].isfinite().all()
    p = torch.tensor([[-3e38, -60.0, -9.0, -0.0, 0.0, 9.0, 60.0, 3e38]], device="cuda").to(BF)
    eye = torch.eye(8, device="cuda", dtype=BF)
    for a, f in (("silu", F.silu), ("gelu", F.gelu), ("relu", torch.relu)):
        want = f(p.double())
        got = linear_act(p, eye, None, a).double()
        torch.testing.assert_close(got, want, rtol=2.0 ** -8, atol=2e-6)


@pytest.mark.gpu
def test_another_stream_and_captured_graphs():
    x, w, wu = rn(300, 64, dev="cuda", dtype=BF), rn(64, 264, dev="cuda", dtype=BF) / 8, rn(64, 264, seed=1, dev="cuda", dtype=BF) / 8
    wd, b, dy = rn(264, 64, dev="cuda", dtype=BF) / 16, rn(264, dev="cuda", dtype=BF), rn(300, 64, seed=2, dev="cuda", dtype=BF)
    leaves = [t.requires_grad_() for t in (x, w, wu, wd, b)]

    def block():
        h = gated_linear(x, w, wu, b, activation="silu", keep="8bit")
        return linear_act(h, wd, residual=x)

    def step():
        y = block()
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
        for _ in range(2):
            step()
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    # (no eager graph of these leaves may live over the capture: autograd would wait for that graph's stream, which
    # ends a capture whatever the operator)
    graphs = []
    for _ in range(2):  # two graphs, whose memory is their own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step()
        graphs.append((g, out))
    with torch.no_grad():
        x.copy_(x.flip(0))
    want2 = step()
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, c) for a, c in zip(out, want2))


@pytest.mark.gpu
def test_few_rows_answer_as_among_many():
    """A token alone, in a batch of few rows and in one of many: other tiles and splits, the same numbers but for fp32 sums."""
    x, w, wu = rn(400, 264, dev="cuda", dtype=BF), rn(264, 520, dev="cuda", dtype=BF) / 16, rn(264, 520, seed=1, dev="cuda", dtype=BF) / 16
    many = gated_linear(x, w, wu, activation="gelu").double()
    for n in (1, 16, 17, 64, 65, 128, 129):
        got = gated_linear(x[:n], w, wu, activation="gelu").double()
        # each is rounded once from sums that differ by 264 units of 2^-23 of their terms
        torch.testing.assert_close(got, many[:n], rtol=2.0 ** -7, atol=1e-4)


def blocks(dev, dtype):
    torch.manual_seed(0)
    plain = MicroTransformerBlock(32, 4, 2).to(dev, dtype)
    fused = MicroTransformerBlock(32, 4, 2, fused=True).to(dev, dtype)
    fused.load_state_dict(plain.state_dict())
    return plain, fused


def test_micro_transformer_with_fused_products_on_the_cpu():
    plain, fused = blocks("cpu", torch.float64)
    x = rn(2, 6, 32).double()
    torch.testing.assert_close(fused(x, 2), plain(x, 2))
    a, b = (torch.autograd.grad(m(x).square().sum(), list(m.parameters())) for m in (plain, fused))
    for p, q in zip(a, b):
        torch.testing.assert_close(p, q)


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [None, "8bit"])
def test_micro_transformer_with_fused_products_on_the_device(keep):
    plain, fused = blocks("cuda", BF)
    fused.keep = keep
    exact = blocks("cuda", torch.float64)[0]
    exact.load_state_dict(plain.state_dict())
    x = rn(3, 50, 32, dev="cuda", dtype=BF)
    want = exact(x.double())
    # the fused block rounds at fewer places than the plain one in bf16: no further from 64 bits than twice its distance
    far = (plain(x).double() - want).norm()
    assert (fused(x).double() - want).norm() <= 2 * far
    grads = lambda m, v: torch.autograd.grad(m(v).double().square().sum(), list(m.parameters()))  # noqa: E731
    for g, p, e in zip(grads(fused, x), grads(plain, x), grads(exact, x.double())):
        assert torch.isfinite(g).all()
        if keep is None:
            assert (g.double() - e).norm() <= 2 * (p.double() - e).norm() + 2.0 ** -8 * e.norm()


def variant(**kw):
    c = DragonConfig(n_layer=2, n_embd=32, n_head=2, mlp_internal_dim_multiplier=4, dropout=0.0, rotary_embedding="rope",
                     initialization="simple_normal", vocab_size=64, sequence_memory_system="mamba3_state_space_duality")
    c.mamba.headdim, c.mamba.chunk_size = 16, 4
    c.latent_reasoning.enabled, c.next_latent_transition.enabled = True, True
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def test_variant_with_the_operators_on_the_cpu():
    t = torch.randint(0, 64, (2, 9), generator=torch.Generator().manual_seed(1))
    a, b = DragonRuntime(variant(), seed=3), DragonRuntime(variant(feed_forward="kernels"), seed=3)
    torch.testing.assert_close(b.forward(t), a.forward(t), rtol=1e-5, atol=1e-6)
    ga, gb = (torch.autograd.grad(m.loss(t, t), [p for p in m.parameters() if p.requires_grad], allow_unused=True) for m in (a, b))
    for p, q in zip(ga, gb):
        assert (p is None) == (q is None)
        if p is not None:
            torch.testing.assert_close(q, p, rtol=1e-4, atol=1e-6)
    h = torch.randn(2, 3, 32)
    torch.testing.assert_close(b.next_latent_prediction(h, h), a.next_latent_prediction(h, h), rtol=1e-5, atol=1e-6)
    with pytest.raises(ValueError):
        variant(feed_forward="triton").validate()
    bad = TrainingConfig()
    bad.training.activation_checkpoints = "4bit"
    with pytest.raises(ValueError):
        bad.validate()
    with pytest.raises(ValueError):
        RuntimeTrainer(variant(), "cpu", activation_checkpoints="4bit")


@pytest.mark.parametrize("kernels", ["torch", "kernels"])
def test_variant_trains_with_activations_in_8_bits_on_the_cpu(kernels):
    train(variant(feed_forward=kernels), "cpu")


def train(cfg, dev):
    t = torch.randint(0, 64, (4, 64), generator=torch.Generator().manual_seed(1))
    full, held = (RuntimeTrainer(cfg, dev, activation_checkpoints=how, seed=5) for how in ("full", "8bit"))
    loss = full.model.loss(t.to(dev), t.to(dev))
    assert torch.equal(held.model.loss(t.to(dev), t.to(dev)), loss)  # the forward pass is the same
    params = lambda tr: [p for p in tr.model.parameters() if p.requires_grad]  # noqa: E731
    a, b = (torch.autograd.grad(tr.model.loss(t.to(dev), t.to(dev)), params(tr), allow_unused=True) for tr in (full, held))
    diff = sum(float((p - q).double().square().sum()) for p, q in zip(a, b) if p is not None)
    size = sum(float(p.double().square().sum()) for p in a if p is not None)
    assert 0 < diff < 0.15 ** 2 * size  # values within 2^-4 of what they were, a few of them in a product
    assert torch.isfinite(held.step(t, t)) and torch.isfinite(held.step(t, t))


@pytest.mark.gpu
def test_variant_with_the_operators_on_the_device():
    t = torch.randint(0, 64, (2, 70), generator=torch.Generator().manual_seed(1)).cuda()
    a, b = DragonRuntime(variant(), device="cuda", seed=3), DragonRuntime(variant(feed_forward="kernels"), device="cuda", seed=3)
    want, got = a.forward(t), b.forward(t)
    # bf16 operands and results (2^-9 each, root mean square less) through two layers of norms
    assert (got - want).norm() <= 0.03 * want.norm()
    st = RuntimeState.new(2)
    parts = [b.forward(t[:, :60], st)] + [b.forward(t[:, i:i + 1], st) for i in range(60, 70)]
    assert (torch.cat(parts, 1) - got).norm() <= 0.03 * got.norm()
    ga, gb = (torch.autograd.grad(m.loss(t, t), [p for p in m.parameters() if p.requires_grad], allow_unused=True) for m in (a, b))
    diff = sum(float((p - q).double().square().sum()) for p, q in zip(ga, gb) if p is not None)
    assert diff < 0.05 ** 2 * sum(float(p.double().square().sum()) for p in ga if p is not None)
    train(variant(feed_forward="kernels"), "cuda")


@pytest.mark.gpu
def test_what_the_products_save_is_held_in_8_bits_too():
    x, w = rn(256, 64, dev="cuda", dtype=BF).requires_grad_(), (rn(64, 512, dev="cuda", dtype=BF) / 8).requires_grad_()
    wd = (rn(512, 64, dev="cuda", dtype=BF) / 16).requires_grad_()

    def run():
        return linear_act(linear_act(x, w, activation="gelu", keep="8bit"), wd)

    def bytes_held(f):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = f()
        return torch.cuda.memory_allocated() - before, y

    def held():
        with activations_in_8bit():
            return run()

    plain, a = bytes_held(run)
    less, b = bytes_held(held)
    assert torch.equal(a, b) and less < plain - 256 * 512 // 2  # the hidden activations: one byte a value and not two
    ga, gb = (torch.autograd.grad(y.float().sum(), (x, w, wd)) for y in (a, b))
    assert torch.equal(ga[0], gb[0]) and torch.equal(ga[1], gb[1])  # x and the weights are leaves
    assert (ga[2] - gb[2]).float().norm() < 2.0 ** -4 * ga[2].float().norm()
