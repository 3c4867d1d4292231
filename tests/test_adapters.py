"""Adapters of many requests beside a shared projection, against the formula in 64 bits."""

import numpy as np
import pytest
import torch

from burn_dragon_b200.ops.adapters import AdapterBatch, adapter_linear

BF = torch.finfo(torch.bfloat16).eps / 2  # relative error of one rounding to bf16 (8 significant bits)


def rows_of(ids, lengths):
    return torch.from_numpy(np.repeat(np.asarray(ids), np.asarray(lengths)))


def formula(x, w, a, b, of, scale):
    """y and what bounds its error, adapter by adapter, every product and sum in 64 bits."""
    x, w, a, b, scale = (t.double() for t in (x, w, a, b, scale))
    M, (H, K, N) = x.shape[0], w.shape
    xh = x[:, None].expand(M, H, K) if x.dim() == 2 else x
    y = torch.einsum("mhk,hkn->mhn", xh, w)
    size = torch.einsum("mhk,hkn->mhn", xh.abs(), w.abs())
    low = torch.zeros_like(y)
    for g in of.unique().tolist():
        if g < 0:
            continue
        rows = of == g
        t = torch.einsum("mhk,hrk->mhr", xh[rows], a[g])
        y[rows] += scale[g] * torch.einsum("mhr,hrn->mhn", t, b[g])
        low[rows] = scale[g] * torch.einsum("mhr,hrn->mhn", t.abs(), b[g].abs())
        t = torch.einsum("mhk,hrk->mhr", xh[rows].abs(), a[g].abs())
        size[rows] += scale[g] * torch.einsum("mhr,hrn->mhn", t, b[g].abs())
    return y, low, size, xh


def gradients(x, w, a, b, of, scale, dy):
    """dx, da, db from the formulas in 64 bits, with the sums of absolute values that bound their errors."""
    x, w, a, b, scale, dy = (v.double() for v in (x, w, a, b, scale, dy))
    M, (H, K, N) = x.shape[0], w.shape
    xh = x[:, None].expand(M, H, K) if x.dim() == 2 else x
    dx, dxe = (torch.einsum("mhn,hkn->mhk", d, v) for d, v in ((dy, w), (dy.abs(), w.abs())))
    da, db, dae, dbe = (torch.zeros_like(v) for v in (a, b, a, b))
    for g in of.unique().tolist():
        if g < 0:
            continue
        rows = of == g
        for absolute, ox, oa, ob in ((False, dx, da, db), (True, dxe, dae, dbe)):
            f = torch.abs if absolute else (lambda v: v)
            u = torch.einsum("mhn,hrn->mhr", f(dy[rows]), f(b[g]))
            t = torch.einsum("mhk,hrk->mhr", f(xh[rows]), f(a[g]))
            ox[rows] += scale[g] * torch.einsum("mhr,hrk->mhk", u, f(a[g]))
            oa[g] = scale[g] * torch.einsum("mhr,mhk->hrk", u, f(xh[rows]))
            ob[g] = scale[g] * torch.einsum("mhr,mhn->hrn", t, f(dy[rows]))
    if x.dim() == 2:
        dx, dxe = dx.sum(1), dxe.sum(1)
    return (dx, dxe), (da, dae), (db, dbe)


def make(ids, lengths, G, H, K, N, r, shared, dev, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    M = int(sum(lengths))
    x = (rn(M, K) if shared else rn(M, H, K)).to(dtype)
    w, a, b = rn(H, K, N) * 0.1, rn(G, H, r, K) * K ** -0.5, rn(G, H, r, N) * 0.2
    scale = torch.rand(G, generator=gen) + 0.5
    return [t.to(dev) for t in (x, w.to(dtype), a.to(dtype), b.to(dtype), scale, rn(M, H, N).to(dtype))]


def within(got, want, bound):
    """|got - want| <= bound everywhere; the bounds are derived, not tuned."""
    assert torch.isfinite(got).all()
    over = (got.double() - want).abs() - bound
    assert over.max() <= 0, f"over the bound by {float(over.max()):.3g} (largest value {float(want.abs().max()):.3g})"


def check(ids, lengths, G, H, K, N, r, shared, train=True):
    x, w, a, b, scale, dy = make(ids, lengths, G, H, K, N, r, shared, "cuda", torch.bfloat16)
    of = rows_of(ids, lengths).cuda()
    batch = AdapterBatch(ids, lengths, G)
    for t in (x, a, b):
        t.requires_grad_(train)
    y = adapter_linear(x, w, a, b, batch, scale)
    want, low, size, _ = formula(x.detach(), w, a.detach(), b.detach(), of, scale)
    # one rounding of y, one of each t, fp32 sums of K + r terms (2^-23 each, chopped sums included)
    acc = (K + 64) * 2.0 ** -23
    within(y.detach(), want, BF * 1.01 * (want.abs() + low) + acc * size)
    if not train:
        return
    got = torch.autograd.grad(y, (x, a, b), dy)
    ref = gradients(x.detach(), w, a.detach(), b.detach(), of, scale, dy)
    terms = (H * N, N + x.shape[0], K + x.shape[0])
    for g, (want, size), n in zip(got, ref, terms):
        # one rounding of the result, one of each u (or t) inside the sum, fp32 sums
        within(g, want, BF * 1.01 * (want.abs() + size) + (n + 64) * 2.0 ** -23 * size)


CASES = [
    # ids, rows, adapters, H, K, N, r, x shared by the heads
    ([0], [1], 1, 1, 64, 64, 16, True),                       # one token
    ([2], [1], 4, 4, 64, 512, 8, True),                       # one token, four heads
    ([-1, -1], [1, 3], 2, 2, 64, 72, 16, True),               # nobody has an adapter
    ([0, -1, 1, 0], [1, 1, 1, 1], 2, 1, 8, 8, 1, True),       # smallest sizes, rank 1
    ([3, 1, 3, 0, -1, 2, 1], [5, 1, 0, 40, 9, 33, 2], 5, 2, 200, 136, 5, True),   # odd sizes, a request of no rows
    (list(range(64)) + [7, 7], [1] * 66, 64, 1, 264, 320, 16, True),              # single tokens, all different
    (list(range(130)), [1] * 130, 130, 1, 128, 256, 24, True),                    # more slots than a tile of rows
    ([0, 1, 2], [127, 1, 129], 3, 2, 192, 128, 32, False),    # tiles that end inside a request, one input per head
    ([1, 0], [300, 213], 3, 3, 136, 72, 64, False),           # full rank width, an adapter that nobody uses
    ([0, 1], [70, 60], 2, 1, 4104, 40, 16, True),             # long reduction, few tiles: split
    ([0, 1, 0], [40, 50, 60], 2, 2, 72, 2056, 33, True),      # wide output, padded rank
    ([1, 3, 0, 2, 1], [301, 1, 499, 64, 36], 4, 2, 256, 9000, 16, True),  # several tiles per CTA, short reduction
    ([0, -1, 1], [700, 300, 36], 2, 3, 72, 6000, 24, True),   # many row tiles of a short reduction, a tile without adapters
    (list(range(40)) * 2, [8] * 80, 40, 2, 64, 8200, 16, False),  # more adapter blocks than projection blocks
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=range(len(CASES)))
def test_forward_and_gradients_on_the_device(case):
    check(*case)


@pytest.mark.gpu
def test_without_heads_and_with_one_scale():
    x, w, a, b, scale, dy = make([0, 1], [3, 20], 2, 1, 96, 104, 8, True, "cuda", torch.bfloat16)
    batch = AdapterBatch([0, 1], [3, 20], 2)
    with_heads = adapter_linear(x, w, a, b, batch, 1.5)
    plain = adapter_linear(x, w[0], a[:, 0], b[:, 0], batch, 1.5)
    assert plain.shape == (23, 104) and torch.equal(plain, with_heads[:, 0])
    assert torch.equal(plain, adapter_linear(x, w[0], a[:, 0], b[:, 0], batch, torch.full((2,), 1.5, device="cuda")))


@pytest.mark.gpu
def test_strided_and_misaligned_inputs_and_another_stream():
    x, w, a, b, scale, _ = make([1, 0], [30, 9], 2, 2, 64, 88, 16, False, "cuda", torch.bfloat16)
    batch = AdapterBatch([1, 0], [30, 9], 2)
    want = adapter_linear(x, w, a, b, batch, scale)
    wide = torch.zeros(39, 2, 64 + 8, dtype=torch.bfloat16, device="cuda")
    wide[:, :, :64] = x
    assert torch.equal(adapter_linear(wide[:, :, :64], w, a, b, batch, scale), want)  # rows of a wider tensor
    odd = torch.zeros(x.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(x.shape).copy_(x)
    assert odd.data_ptr() % 16 and torch.equal(adapter_linear(odd, w, a, b, batch, scale), want)
    turned = x.transpose(0, 2).contiguous().transpose(0, 2)
    assert torch.equal(adapter_linear(turned, w.transpose(1, 2).contiguous().transpose(1, 2), a, b, batch, scale), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = adapter_linear(x, w, a, b, batch, scale)
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_rows_do_not_depend_on_the_batch_around_them():
    """A request alone answers as it does among others, bit for bit, and twice the same."""
    ids, lengths = [0, 2, 1, -1], [3, 200, 50, 7]
    x, w, a, b, scale, _ = make(ids, lengths, 3, 1, 128, 256, 16, True, "cuda", torch.bfloat16)
    y = adapter_linear(x, w, a, b, AdapterBatch(ids, lengths, 3), scale)
    assert torch.equal(y, adapter_linear(x, w, a, b, AdapterBatch(ids, lengths, 3), scale))
    without = adapter_linear(x, w, a, b, AdapterBatch([-1] * 4, lengths, 3), scale)
    assert torch.equal(y[253:], without[253:]) and not torch.equal(y[:253], without[:253])


@pytest.mark.gpu
def test_a_not_finite_row_stays_in_its_row():
    """Other rows of the tile, and other adapters, are not touched by infinities or NaN of one request."""
    ids, lengths = [0, 1, 0], [2, 1, 5]
    x, w, a, b, scale, _ = make(ids, lengths, 2, 1, 64, 64, 16, True, "cuda", torch.bfloat16)
    batch = AdapterBatch(ids, lengths, 2)
    want = adapter_linear(x, w, a, b, batch, scale)
    x[2] = float("nan")
    got = adapter_linear(x, w, a, b, batch, scale)
    keep = torch.arange(8, device="cuda") != 2
    assert torch.equal(got[keep], want[keep]) and got[2].isnan().all()


@pytest.mark.gpu
def test_gradients_against_differences():
    """The function is linear in x and in b: a central difference in 64 bits is exact up to rounding."""
    ids, lengths, G, H, K, N, r = [0, 1, -1, 0], [4, 9, 2, 5], 2, 2, 64, 72, 8
    x, w, a, b, scale, dy = make(ids, lengths, G, H, K, N, r, True, "cuda", torch.bfloat16)
    of = rows_of(ids, lengths).cuda()
    for t in (x, a, b):
        t.requires_grad_(True)
    got = torch.autograd.grad(adapter_linear(x, w, a, b, AdapterBatch(ids, lengths, G), scale), (x, a, b), dy)
    args = [t.detach().double() for t in (x, a, b)]
    sizes = gradients(x.detach(), w, a.detach(), b.detach(), of, scale, dy)
    gen = torch.Generator(device="cuda").manual_seed(3)
    for i in range(3):
        v = torch.randn(args[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        f = []
        for sign in (1.0, -1.0):
            moved = list(args)
            moved[i] = moved[i] + sign * 0.25 * v
            f.append((formula(moved[0], w, moved[1], moved[2], of, scale)[0] * dy.double()).sum())
        slope = (f[0] - f[1]) / 0.5
        bound = ((BF * 1.01 * (sizes[i][0].abs() + sizes[i][1]) + 1024 * 2.0 ** -23 * sizes[i][1]) * v.abs()).sum()
        assert (slope - (got[i].double() * v).sum()).abs() <= bound


def test_cpu_path_matches_formula_and_gradcheck():
    ids, lengths, G, H, K, N, r = [1, -1, 0, 1], [2, 1, 3, 0], 2, 2, 8, 16, 3
    for shared in (True, False):
        x, w, a, b, scale, _ = make(ids, lengths, G, H, K, N, r, shared, "cpu", torch.float64)
        batch = AdapterBatch(ids, lengths, G, device="cpu")
        want = formula(x, w, a, b, rows_of(ids, lengths), scale)[0]
        assert torch.allclose(adapter_linear(x, w, a, b, batch, scale.double()), want, atol=1e-12)
        for t in (x, a, b):
            t.requires_grad_(True)
        assert torch.autograd.gradcheck(lambda x, a, b: adapter_linear(x, w, a, b, batch, scale.double()), (x, a, b))


@pytest.mark.parametrize("seed", range(6))
def test_plan_covers_every_row_once(seed):
    rng = np.random.default_rng(seed)
    G, R = int(rng.integers(1, 20)), int(rng.integers(0, 40))
    ids, lengths = rng.integers(-1, G, R), rng.integers(0, 60, R)
    batch = AdapterBatch(ids, lengths, G, device="cpu")
    M, G, tiles, n_slots, n_rows, n_chunks, per = batch.dims
    of = np.repeat(ids, lengths)
    flat = batch.plan.numpy()
    row_adapter, row_slot, tile_ptr, slots, order, chunk, group, by_size = np.split(
        flat, np.cumsum([M, M, tiles + 1, n_slots, n_rows, 3 * n_chunks, G + 1]))
    assert (row_adapter == of).all() and group.size == G + 1
    for m in range(M):
        if of[m] < 0:
            assert row_slot[m] == -1
        else:
            lo, hi = tile_ptr[m // 128], tile_ptr[m // 128 + 1]
            assert 0 <= row_slot[m] < hi - lo and slots[lo + row_slot[m]] == of[m]
    assert sorted(order) == list(np.flatnonzero(of >= 0))
    seen = np.zeros(n_rows, int)
    for start, count, g in chunk.reshape(-1, 3):
        assert 1 <= count <= per and (of[order[start:start + count]] == g).all()
        seen[start:start + count] += 1
    assert (seen == 1).all()
    for g in range(G):
        assert (of[order[group[g]:group[g + 1]]] == g).all()
    assert group[G] == n_rows
    assert sorted(by_size) == list(range(G)) and (np.diff(np.diff(group)[by_size]) <= 0).all()


def test_refusals():
    batch = AdapterBatch([0, 1], [2, 3], 2, device="cpu")
    x, w, a, b, scale, _ = make([0, 1], [2, 3], 2, 2, 16, 24, 4, True, "cpu", torch.float32)
    with pytest.raises(ValueError, match="adapter ids"):
        AdapterBatch([2], [1], 2, device="cpu")
    with pytest.raises(ValueError, match="adapter ids"):
        AdapterBatch([-2], [1], 2, device="cpu")
    with pytest.raises(ValueError, match="requests"):
        AdapterBatch([0], [1, 2], 2, device="cpu")
    with pytest.raises(ValueError, match="fewer than 0"):
        AdapterBatch([0], [-1], 2, device="cpu")
    with pytest.raises(ValueError, match="does not fit"):
        adapter_linear(x[:4], w, a, b, batch, scale)
    with pytest.raises(ValueError, match="do not fit"):
        adapter_linear(x, w, a, b[:, :, :3], batch, scale)
    with pytest.raises(ValueError, match="planned for"):
        adapter_linear(x, w, a[:1], b[:1], batch, 1.0)
    with pytest.raises(ValueError, match="one value per adapter"):
        adapter_linear(x, w, a, b, batch, torch.ones(3))
    with pytest.raises(ValueError, match="frozen"):
        adapter_linear(x, w.clone().requires_grad_(True), a, b, batch, scale)
    with pytest.raises(ValueError, match="without heads"):
        adapter_linear(x, w[0], a, b, batch, scale)


@pytest.mark.gpu
def test_refusals_on_the_device():
    batch = AdapterBatch([0], [5], 2)
    x, w, a, b, scale, _ = make([0], [5], 2, 2, 16, 24, 4, True, "cuda", torch.bfloat16)
    with pytest.raises(TypeError, match="bf16"):
        adapter_linear(x.float(), w, a, b, batch, scale)
    with pytest.raises(ValueError, match="multiples of 8"):
        adapter_linear(x[:, :12].contiguous(), w[:, :12].contiguous(), a[..., :12].contiguous(), b, batch, scale)
    with pytest.raises(ValueError, match="rank"):
        adapter_linear(x, w, a.repeat(1, 1, 17, 1), b.repeat(1, 1, 17, 1), batch, scale)
    with pytest.raises(ValueError, match="one device"):
        adapter_linear(x, w.cpu(), a, b, batch, scale)
    with pytest.raises(ValueError, match="one device"):
        adapter_linear(x, w, a, b, AdapterBatch([0], [5], 2, device="cpu"), scale)
