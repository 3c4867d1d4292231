"""linear_act and gated_linear against their formulas in 64 bits.

Inputs are small multiples of powers of two, so that every pre-activation is exact in fp32 in any order of summation: what a
relu passes, what 16 bits and 8 bits hold is then the same on both sides, and the bounds count roundings only.
"""

import math

import pytest
import torch

from burn_dragon_b200.ops.act8 import pack_activation
from burn_dragon_b200.ops.feed_forward import gated_linear, linear_act

ACTS = ("none", "relu", "silu", "gelu")
FUNCTION = 2.0 ** -19  # exp and erf in fp32 and what is made of them: a few units of 2^-23 relative to 1


def act(p, kind):
    """The activation and its derivative in 64 bits."""
    if kind == "relu":
        return p.clamp_min(0), (p > 0).double()
    if kind == "silu":
        s = torch.sigmoid(p)
        return p * s, s + p * s * (1 - s)
    if kind == "gelu":
        cdf = 0.5 * torch.erfc(-p / math.sqrt(2))
        return p * cdf, cdf + p * torch.exp(-p * p / 2) / math.sqrt(2 * math.pi)
    return p, torch.ones_like(p)


def seen(p, keep, dtype):
    if keep == "16bit":
        return p.to(dtype).double()
    return pack_activation(p.float()).unpack().double() if keep == "8bit" else p


def small(gen, shape, step, dtype, dev):
    return (torch.randint(-3, 4, shape, generator=gen).float() * step).to(dtype).to(dev)


def within(got, want, bound, what):
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    over = ((got.double() - want).abs() - bound).max() if got.numel() else torch.zeros(())
    assert over <= 0, f"{what}: over the bound by {float(over):.3g} (largest value {float(want.abs().max()):.3g})"


def sums(n):
    """What an fp32 sum of n terms loses relative to the sum of their sizes, chopped additions included."""
    return (n + 64) * 2.0 ** -22


def check_linear(M, K, N, kind, bias, residual, turned, dtype, keep, dev="cuda", train=True):
    gen = torch.Generator().manual_seed(M + 3 * K + 7 * N)
    half = torch.finfo(dtype).eps / 2 * 1.01
    x = small(gen, (M, K), 0.5, dtype, dev)
    w = small(gen, (N, K) if turned else (K, N), 2.0 ** -max(2, round(math.log2(max(K, 1)) / 2) + 1), dtype, dev)
    w = w.t() if turned else w
    b = None if bias is None else bias if isinstance(bias, float) else small(gen, (N,), 0.25, bias, dev)
    r = small(gen, (M, N), 0.25, dtype, dev) if residual else None
    dy = small(gen, (M, N), 0.5, dtype, dev)
    leaves = [t for t in (x, w, b, r) if isinstance(t, torch.Tensor)]
    for t in leaves:
        t.requires_grad_(train)
    y = linear_act(x, w, b, kind, residual=r, keep=keep)
    assert y.dtype == dtype
    xd, wd = x.detach().double(), w.detach().double()
    p = xd @ wd + (0 if b is None else b if isinstance(b, float) else b.detach().double())
    f, _ = act(p, kind)
    want = f + (0 if r is None else r.detach().double())
    within(y.detach(), want, half * want.abs() + FUNCTION * (1 + f.abs()) + (2.0 ** -23 * want.abs()), "y")
    if not train:
        return
    got = dict(zip(("x", "w", "b", "r") if isinstance(b, torch.Tensor) else ("x", "w", "r"),
                   torch.autograd.grad(y, leaves, dy)))
    d = dy.double()
    dp = d * act(seen(p, keep, dtype), kind)[1]
    e = half * dp.abs() + 4 * FUNCTION * d.abs()  # one rounding of dp, and the derivative's own error
    want, size, off = dp @ wd.t(), dp.abs() @ wd.abs().t(), e @ wd.abs().t()
    within(got["x"], want, half * want.abs() + off + sums(N) * size, "dx")
    want, size, off = xd.t() @ dp, xd.abs().t() @ dp.abs(), xd.abs().t() @ e
    within(got["w"], want, half * want.abs() + off + sums(M) * size, "dw")
    if isinstance(b, torch.Tensor):
        want = dp.sum(0)
        within(got["b"], want, torch.finfo(b.dtype).eps / 2 * 1.01 * want.abs() + 4 * FUNCTION * d.abs().sum(0)
               + sums(M) * dp.abs().sum(0), "db")
    if r is not None:
        assert torch.equal(got["r"], dy)


BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
LINEAR = [
    # M, K, N, activation, bias, residual, turned, type, keep
    (1, 8, 8, "none", None, False, False, BF, None),
    (1, 64, 256, "gelu", BF, False, True, BF, "16bit"),
    (1, 1, 1, "relu", F32, True, False, HF, "8bit"),              # smallest, padded
    (3, 72, 40, "silu", 0.25, False, False, BF, "8bit"),
    (5, 13, 7, "gelu", F32, True, True, BF, "recompute"),         # nothing is a multiple of anything
    (33, 64, 96, "relu", None, True, False, HF, "recompute"),
    (48, 4104, 40, "none", HF, True, False, HF, None),            # long reduction, few tiles: split
    (64, 2056, 72, "silu", BF, True, True, BF, "8bit"),           # split, with everything in the joining kernel
    (100, 3000, 136, "gelu", None, False, False, BF, "recompute"),
    (128, 64, 64, "relu", BF, False, False, BF, "16bit"),
    (129, 136, 264, "gelu", BF, True, False, BF, "16bit"),        # two CTAs, ragged everywhere
    (257, 64, 520, "silu", F32, False, True, HF, "8bit"),
    (300, 200, 1001, "gelu", BF, True, False, BF, "8bit"),        # padded columns
    (700, 256, 2056, "relu", F32, False, True, BF, "recompute"),
    (1000, 72, 6000, "gelu", HF, False, False, HF, "16bit"),      # several tiles a CTA
    (2050, 520, 640, "none", BF, False, True, BF, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", LINEAR, ids=range(len(LINEAR)))
def test_linear_on_the_device(case):
    check_linear(*case)
    check_linear(*case, train=False)


@pytest.mark.parametrize("case", LINEAR[:7], ids=range(7))
def test_linear_on_the_cpu(case):
    check_linear(*case, dev="cpu")


def check_gated(M, H, K, N, kind, up, z, per_head, bias, turned, dtype, keep, dev="cuda", train=True):
    gen = torch.Generator().manual_seed(M + 3 * K + 7 * N + H)
    half = torch.finfo(dtype).eps / 2 * 1.01
    heads = H > 0
    Hn = max(H, 1)
    step = 2.0 ** -max(2, round(math.log2(max(K, 1)) / 2) + 1)
    x = small(gen, (M, H, K) if per_head and heads else (M, K), 0.5, dtype, dev)
    zz = small(gen, (M, H, K) if heads and z == "heads" else (M, K), 0.5, dtype, dev) if z else None
    ws = []
    for i in range(2):
        w = small(gen, (Hn, N, K) if turned[i] else (Hn, K, N), step, dtype, dev)
        w = w.transpose(1, 2) if turned[i] else w
        ws.append(w if heads else w[0])
    wg, wu = ws
    bg = bu = None
    if isinstance(bias, float):
        bg, bu = bias, -bias
    elif bias is not None:
        bg, bu = (small(gen, (H, N) if heads else (N,), 0.25, bias, dev) for _ in range(2))
    dy = small(gen, (M, H, N) if heads else (M, N), 0.5, dtype, dev)
    leaves = [t for t in (x, zz, wg, wu, bg, bu) if isinstance(t, torch.Tensor)]
    names = [n for n, t in zip(("x", "z", "wg", "wu", "bg", "bu"), (x, zz, wg, wu, bg, bu)) if isinstance(t, torch.Tensor)]
    for t in leaves:
        t.requires_grad_(train)
    y = gated_linear(x, wg, wu, bg, bu, z=zz, activation=kind, up_activation=up, keep=keep)
    assert y.dtype == dtype and y.shape == dy.shape

    def wide(t):  # [M, Hn, K]
        t = t.detach().double()
        return t if t.dim() == 3 else t[:, None].expand(M, Hn, K)

    def column(b):
        return 0 if b is None else b if isinstance(b, float) else b.detach().double().reshape(Hn, N)

    xd, zd = wide(x), wide(x if zz is None else zz)
    wgd, wud = (w.detach().double().reshape(Hn, K, N) for w in (wg, wu))
    g, u = torch.einsum("mhk,hkn->mhn", xd, wgd) + column(bg), torch.einsum("mhk,hkn->mhn", zd, wud) + column(bu)
    (f, _), (h, _) = act(g, kind), act(u, up)
    want = (f * h).reshape(dy.shape)
    within(y.detach(), want, half * want.abs() + (FUNCTION * (1 + f.abs()) * h.abs() + 2.0 ** -22 * (f * h).abs()).reshape(dy.shape),
           "y")
    if not train:
        return
    got = dict(zip(names, torch.autograd.grad(y, leaves, dy)))
    d = dy.double().reshape(M, Hn, N)
    (f, df), (h, dh) = act(seen(g, keep, dtype), kind), act(seen(u, keep, dtype), up)
    dg, du = d * h * df, d * f * dh
    eg = half * dg.abs() + 4 * FUNCTION * (d * h).abs() + 2.0 ** -21 * dg.abs()
    eu = half * du.abs() + 4 * FUNCTION * (d * dh).abs() * (1 + f.abs()) + 2.0 ** -21 * du.abs()
    back = lambda t, w: torch.einsum("mhn,hkn->mhk", t, w)  # noqa: E731
    parts = {"x": [(dg, eg, wgd)] + ([(du, eu, wud)] if zz is None else []), "z": [(du, eu, wud)]}
    for n, t in (("x", x), ("z", zz)):
        if t is None:
            continue
        want = sum(back(a, w) for a, _, w in parts[n])
        size = sum(back(a.abs(), w.abs()) for a, _, w in parts[n])
        off = sum(back(e, w.abs()) for _, e, w in parts[n])
        terms = N * len(parts[n])
        if t.dim() == 2:
            want, size, off, terms = want.sum(1), size.sum(1), off.sum(1), terms * Hn
        within(got[n], want, half * want.abs() + off + sums(terms) * size, "d" + n)
    for n, t, a, e in (("wg", xd, dg, eg), ("wu", zd, du, eu)):
        want, size, off = (torch.einsum("mhk,mhn->hkn", p, q) for p, q in ((t, a), (t.abs(), a.abs()), (t.abs(), e)))
        like = got[n].shape
        within(got[n], want.reshape(like), (half * want.abs() + off + sums(M) * size).reshape(like), "d" + n)
    for n, b, a, e in (("bg", bg, dg, eg), ("bu", bu, du, eu)):
        if isinstance(b, torch.Tensor):
            want = a.sum(0).reshape(b.shape)
            bound = torch.finfo(b.dtype).eps / 2 * 1.01 * want.abs() + (e + sums(M) * a.abs()).sum(0).reshape(b.shape)
            within(got[n], want, bound, "d" + n)


NO, YES = (False, False), (True, True)
GATED = [
    # M, heads (0: none), K, N, activation, up, z, x per head, bias, turned, type, keep
    (1, 4, 64, 512, "relu", "relu", "heads", False, None, NO, BF, "recompute"),
    (1, 0, 8, 8, "silu", "none", None, False, None, NO, BF, "16bit"),
    (2, 0, 5, 3, "gelu", "none", "shared", False, F32, NO, HF, "8bit"),                # padded
    (37, 2, 72, 40, "silu", "none", "heads", True, BF, YES, BF, "8bit"),
    (64, 4, 64, 512, "relu", "relu", "heads", False, -0.25, NO, BF, "recompute"),
    (20, 0, 4104, 72, "gelu", "none", None, False, BF, NO, BF, "8bit"),                 # split
    (90, 2, 2056, 40, "silu", "relu", "shared", False, HF, YES, HF, "16bit"),           # split
    (70, 0, 3000, 136, "gelu", "none", None, False, None, NO, BF, "recompute"),        # split, also when computed again
    (129, 2, 136, 264, "gelu", "none", "heads", False, BF, NO, BF, "16bit"),            # two CTAs, ragged
    (300, 3, 64, 200, "silu", "relu", None, False, F32, YES, HF, "8bit"),               # x shared by heads and projections
    (515, 2, 64, 328, "relu", "none", None, True, BF, NO, BF, "recompute"),
    (260, 0, 328, 1003, "silu", "none", None, False, BF, (False, True), BF, "8bit"),   # padded, weights laid out differently
    (1100, 4, 64, 2048, "relu", "relu", "heads", False, F32, NO, BF, "recompute"),      # several tiles a CTA
    (600, 0, 1024, 1000, "silu", "none", "shared", False, None, (True, False), HF, "16bit"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", GATED, ids=range(len(GATED)))
def test_gated_on_the_device(case):
    check_gated(*case)
    check_gated(*case, train=False)


@pytest.mark.parametrize("case", GATED[:5], ids=range(5))
def test_gated_on_the_cpu(case):
    check_gated(*case, dev="cpu")
