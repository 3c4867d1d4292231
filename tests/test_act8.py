"""Activations in 8 bits against the definition in 64 bits, and their use by autograd."""

import pytest
import torch

from burn_dragon_b200.ops.act8 import PackedActivation, activations_in_8bit, pack_activation

BLOCK = 32


def definition(x):
    """The values that x's codes stand for, run by run, in 64 bits."""
    flat = x.double().reshape(-1, x.shape[-1])
    out = torch.empty_like(flat)
    for r, row in enumerate(flat):
        for c in range(0, row.numel(), BLOCK):
            v = row[c:c + BLOCK]
            fine = v.isfinite()
            top = float(v[fine].abs().max()) if fine.any() else 0.0
            e = -126
            while top > 448 * 2.0 ** e:
                e += 1
            u = v / 2.0 ** e
            exponent = torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -6)))
            grid = torch.exp2(exponent - 3)
            out[r, c:c + BLOCK] = torch.where(fine, torch.round(u / grid) * grid * 2.0 ** e, float("nan"))
    top = torch.finfo(x.dtype).max
    return out.clamp(-top, top).to(x.dtype).view(x.shape)


CASES = [((1, 1), 1.0), ((3, 31), 1.0), ((2, 32), 1e-3), ((5, 33), 1e4), ((7, 100), 1.0), ((2, 3, 64), 300.0), ((1, 1000), 1.0),
         ((40, 257), 1e-30), ((9, 96), 1e-6)]


def values(shape, size, dtype, dev):
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(*shape, generator=g) * torch.exp2(4 * torch.randn(*shape[:-1], 1, generator=g)) * size
    return x.clamp(-6e4, 6e4).to(dtype).to(dev)


def check(dev):
    for shape, size in CASES:
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            x = values(shape, size, dtype, dev)
            packed = pack_activation(x)
            got = packed.unpack()
            assert got.dtype == dtype and got.shape == x.shape
            torch.testing.assert_close(got.cpu(), definition(x.cpu()), rtol=0, atol=0)
            assert packed.nbytes == x.numel() + x.numel() // x.shape[-1] * -(-x.shape[-1] // BLOCK)


def test_values_on_the_cpu():
    check("cpu")


@pytest.mark.gpu
def test_values_on_the_device():
    check("cuda")


def odd_values(dtype):
    top = torch.finfo(dtype).max
    x = torch.zeros(6, 40, dtype=dtype)
    x[0, 3], x[0, 35] = float("inf"), 2.0
    x[1, :5] = torch.tensor([float("nan"), -float("inf"), 1.0, -3.0, -0.0], dtype=dtype)
    x[2, 0], x[2, 1] = top, -top
    x[3] = float("nan")
    x[4, 7], x[4, 8] = 448.0, 2.0 ** -10  # the largest code, and half the smallest: to even, 0
    x[5, :3] = torch.tensor([torch.finfo(dtype).smallest_normal, torch.finfo(dtype).tiny / 2, -torch.finfo(dtype).tiny], dtype=dtype)
    return x


def check_odd(dev):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = odd_values(dtype).to(dev)
        got = pack_activation(x).unpack().cpu()
        torch.testing.assert_close(got, definition(x.cpu()), rtol=0, atol=0, equal_nan=True)
        assert got[0].isnan().sum() == 1 and got[1].isnan().sum() == 2 and got[3].isnan().all()
        assert got[2].isfinite().all() and float(got[2, 0]) == min(torch.finfo(dtype).max, float(got[2, 0]))


def test_values_that_are_not_finite_and_limits_on_the_cpu():
    check_odd("cpu")


@pytest.mark.gpu
def test_values_that_are_not_finite_and_limits_on_the_device():
    check_odd("cuda")


def check_layouts(dev):
    x = values((12, 70), 1.0, torch.float32, dev)
    turned = x.t().contiguous().t()
    want = pack_activation(x).unpack()
    assert torch.equal(pack_activation(turned).unpack(), want)
    wide = torch.zeros(12, 80, device=dev)
    wide[:, 5:75] = x
    assert torch.equal(pack_activation(wide[:, 5:75]).unpack(), want)
    odd = torch.zeros(x.numel() + 1, device=dev)[1:].view(x.shape).copy_(x)
    assert torch.equal(pack_activation(odd).unpack(), want)
    for shape in ((0, 5), (5, 0), (0,)):
        assert pack_activation(torch.zeros(shape, device=dev)).unpack().shape == shape
    assert float(pack_activation(torch.tensor(3.0, device=dev)).unpack()) == 3.0
    with pytest.raises(TypeError):
        pack_activation(torch.zeros(4, dtype=torch.float64, device=dev))


def test_layouts_and_refusals_on_the_cpu():
    check_layouts("cpu")


@pytest.mark.gpu
def test_layouts_and_refusals_on_the_device():
    check_layouts("cuda")


def check_autograd(dev):
    g = torch.Generator().manual_seed(0)
    w1 = torch.randn(64, 96, generator=g).to(dev).requires_grad_(True)
    w2 = torch.randn(96, 64, generator=g).to(dev).requires_grad_(True)
    x = torch.randn(70, 64, generator=g).to(dev).requires_grad_(True)
    saved = []

    def layer(x):
        h = torch.relu(x @ w1)
        return (h * torch.sigmoid(h)) @ w2

    with activations_in_8bit():
        y = layer(x)
    saved = y.grad_fn._saved_self  # the last product's input, as the backward pass will see it
    h = torch.relu((x @ w1).detach())
    assert torch.equal(saved, pack_activation(h * torch.sigmoid(h)).unpack())
    assert torch.equal(y, layer(x))
    got = torch.autograd.grad(y.square().sum(), (w1, w2, x))
    # by hand: every saved activation read back from 8 bits; the parameters and x as they are
    h8, s8 = (pack_activation(t).unpack() for t in (h, torch.sigmoid(h)))
    p8 = pack_activation(h * torch.sigmoid(h)).unpack()
    dy = 2 * y.detach()
    dp = dy @ w2.detach().t()
    dh = dp * s8 + dp * h8 * s8 * (1 - s8)
    dh = dh * (h8 > 0)
    for a, b in zip(got, (x.detach().t() @ dh, p8.t() @ dy, dh @ w1.detach().t())):
        # the same fp32 products in another order: 96 terms at most
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4 * float(b.abs().max()))


def test_autograd_holds_8_bits_on_the_cpu():
    check_autograd("cpu")


@pytest.mark.gpu
def test_autograd_holds_8_bits_on_the_device():
    check_autograd("cuda")


def test_what_stays_as_it_is():
    w = torch.randn(64, 64, requires_grad=True)
    low = w.to(torch.bfloat16)
    x = torch.randn(100, 64, requires_grad=True)
    with activations_in_8bit(min_values=1, exclude=[low]):
        y = x.to(torch.bfloat16) @ low
        z = x.t() @ x
    assert torch.equal(y.grad_fn._saved_mat2, low)
    assert torch.equal(z.grad_fn._saved_mat2, x)  # a leaf, and above a view of one
    with activations_in_8bit(min_values=1):
        n = (x * 2).norm(dim=-1, keepdim=True)  # rows of one value
        m = n * n
    assert torch.equal(m.grad_fn._saved_self, n)
    assert isinstance(pack_activation(x), PackedActivation) and not pack_activation(x).unpack().requires_grad
