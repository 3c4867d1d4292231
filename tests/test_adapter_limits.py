"""Where adapter_linear must refuse, keep requests apart or give an empty answer."""

import pytest
import torch

from burn_dragon_b200.ops.adapters import AdapterBatch, adapter_linear


def make(M, G=2, H=2, K=16, N=24, r=4, dev="cpu", dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen).to(dev, dtype)  # noqa: E731
    return rn(M, K), rn(H, K, N) * 0.1, rn(G, H, r, K) * K ** -0.5, rn(G, H, r, N) * 0.2


def test_a_plan_of_another_device_is_refused():
    """The plan's indexes decide what is read and written: it has to lie where the operands do."""
    x, w, a, b = make(5)
    elsewhere = AdapterBatch([0, 1], [2, 3], 2, device="meta")
    with pytest.raises(ValueError, match="one device"):
        adapter_linear(x, w, a, b, elsewhere)
    with pytest.raises(ValueError, match="one device"):
        adapter_linear(x, w.to("meta"), a, b, AdapterBatch([0, 1], [2, 3], 2, device="cpu"))


@pytest.mark.gpu
def test_the_binding_refuses_a_plan_of_another_device():
    from burn_dragon_b200 import _ext
    from burn_dragon_b200.ops.gemm import error_word

    x, w, a, b = make(5, dev="cuda", dtype=torch.bfloat16)
    batch = AdapterBatch([0, 1], [2, 3], 2, device="cpu")
    mod, err = _ext.load(), error_word(x.device)
    assert mod.adapter_direct(x, w, a, b, batch.plan, batch.dims, None, 1.0, err) is None
    with pytest.raises(RuntimeError, match="operands' GPU"):
        mod.adapter_forward(x, w, a, b, batch.plan, batch.dims, None, 1.0, err)


LAYOUTS = [
    # ids, rows, adapters, H, K, N, r, x shared: several requests to a tile
    ([0, 1, -1, 2, 0], [3, 2, 4, 5, 1], 3, 2, 64, 72, 16, True),            # one block of adapters
    (list(range(9)) + [-1, 1], [1] * 11, 9, 1, 128, 264, 8, True),          # several blocks, single tokens
    ([2, 1, 0, -1], [100, 20, 60, 9], 3, 2, 72, 136, 33, False),            # one slot a block, two tiles
    (list(range(20)) + [-1] * 3, [2] * 23, 20, 1, 8200, 40, 16, True),      # a reduction in parts
    ([0, 1, 2, -1, 1], [30, 40, 50, 7, 9], 3, 4, 128, 520, 24, True),       # two slots a block, dx sums the heads
]


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["a", "b", "one of b"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("layout", LAYOUTS, ids=range(len(LAYOUTS)))
def test_a_not_finite_adapter_stays_with_its_rows(layout, value, where):
    """Rows of other adapters, rows without one and the other adapters' gradients are what they are beside a finite
    adapter, bit for bit; the adapter's own rows are not finite where the formula's are not."""
    ids, lengths, G, H, K, N, r, shared = layout
    M = sum(lengths)
    gen = torch.Generator().manual_seed(4)
    rn = lambda *s: torch.randn(*s, generator=gen).to("cuda", torch.bfloat16)  # noqa: E731
    x, w = (rn(M, K) if shared else rn(M, H, K)), rn(H, K, N) * 0.1
    a, b, dy = rn(G, H, r, K) * K ** -0.5, rn(G, H, r, N) * 0.2, rn(M, H, N)
    batch = AdapterBatch(ids, lengths, G)
    of = batch.adapter_of_row()

    def run(a, b):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, a, b)]
        y = adapter_linear(leaves[0], w, leaves[1], leaves[2], batch, 0.7)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    want = run(a, b)
    bad = (a if where == "a" else b).clone()
    if where == "one of b":
        bad[1, H - 1, r - 1, N - 3] = value
    else:
        bad[1, H - 1] = value
    got = run(bad, b) if where == "a" else run(a, bad)
    other, rest = of != 1, torch.arange(G, device="cuda") != 1
    assert torch.equal(got[0][other], want[0][other]) and torch.equal(got[1][other], want[1][other])
    assert torch.equal(got[2][rest], want[2][rest]) and torch.equal(got[3][rest], want[3][rest])
    assert not got[0][of == 1].isfinite().all()
    if where == "one of b":  # only its column of y
        columns = torch.ones(H, N, dtype=torch.bool, device="cuda")
        columns[H - 1, N - 3] = False
        assert torch.equal(got[0][:, columns], want[0][:, columns])
        assert not got[0][of == 1][:, H - 1, N - 3].isfinite().any()
    else:
        assert not got[0][of == 1][:, H - 1].isfinite().any()


@pytest.mark.gpu
def test_an_infinite_t_gives_the_formulas_infinity():
    """Ranks are padded to 16, 32 or 64: what pads them adds nothing to an infinite row, not 0 * inf."""
    x, w, a, b = make(6, G=1, H=1, K=64, N=64, r=5, dev="cuda", dtype=torch.bfloat16)
    x, a, b = x.abs(), a.abs(), b.abs()
    a[0, 0, 4, 0] = float("inf")
    y = adapter_linear(x, w, a, b, AdapterBatch([0], [6], 1))
    keep = (x[:, :1] > 0) & (b[0, 0, 4] > 0)
    assert (y[:, 0][keep] == float("inf")).all()


@pytest.mark.gpu
def test_the_gradient_of_an_unused_adapter_is_zero_whatever_its_scale():
    x, w, a, b = make(6, G=3, H=1, K=64, N=64, dev="cuda", dtype=torch.bfloat16)
    scale = torch.tensor([1.0, float("nan"), 2.0], device="cuda")
    a.requires_grad_(True), b.requires_grad_(True)
    y = adapter_linear(x, w, a, b, AdapterBatch([0, 2], [2, 4], 3), scale)
    for g in torch.autograd.grad(y, (a, b), torch.ones_like(y)):
        assert (g[1] == 0).all() and g.isfinite().all()


@pytest.mark.gpu
def test_derivatives_that_the_kernels_do_not_have_are_refused():
    """A tangent or a gradient of the scale must not disappear."""
    import torch.autograd.forward_ad as fwd

    x, w, a, b = make(5, dev="cuda", dtype=torch.bfloat16)
    batch = AdapterBatch([0, 1], [2, 3], 2)
    scale = torch.ones(2, device="cuda")
    with fwd.dual_level():
        for i in range(4):
            args = [x, w, a, b]
            args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                adapter_linear(*args, batch, scale)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            adapter_linear(x, w, a, b, batch, fwd.make_dual(scale, scale))
        adapter_linear(x, w, a, b, batch, scale)
    scale.requires_grad_(True)
    with pytest.raises(ValueError, match="scale is a constant"):
        adapter_linear(x, w, a, b, batch, scale)
    with torch.no_grad():
        adapter_linear(x, w, a, b, batch, scale)


@pytest.mark.parametrize("dev,dtype", [("cpu", torch.float32), pytest.param("cuda", torch.bfloat16, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("ids,lengths", [([], []), ([0], [0]), ([-1, -1], [2, 1])], ids=("no request", "no rows", "no adapters"))
@pytest.mark.parametrize("heads", [True, False])
def test_gradients_where_no_row_has_an_adapter(ids, lengths, heads, dev, dtype):
    """Zeros for a and b, and an empty gradient of no rows: a training step may hold such a batch."""
    x, w, a, b = make(sum(lengths), H=1, dev=dev, dtype=dtype)
    w, a, b = (w, a, b) if heads else (w[0], a[:, 0], b[:, 0])
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, a, b)]
    y = adapter_linear(leaves[0], w, leaves[1], leaves[2], AdapterBatch(ids, lengths, 2, device=dev))
    dx, da, db = torch.autograd.grad(y.sum(), leaves)
    assert y.shape == ((x.shape[0], 1, 24) if heads else (x.shape[0], 24)) and dx.shape == x.shape
    assert (da == 0).all() and (db == 0).all() and da.shape == a.shape and db.shape == b.shape
    if x.shape[0]:
        want = w.double().sum(-1).expand(x.shape)  # one rounding of the result, fp32 sums
        assert ((dx.double() - want).abs() <= torch.finfo(dtype).eps * w.double().abs().sum(-1)).all()
    with torch.no_grad():
        assert not adapter_linear(*[leaves[0], w, *leaves[1:]], AdapterBatch(ids, lengths, 2, device=dev)).requires_grad


@pytest.mark.gpu
def test_adapters_at_odd_addresses_and_strides():
    """a and b that do not start on 16 bytes (parts of one buffer) or are not contiguous are copied, as x is."""
    x, w, a, b = make(9, G=3, H=2, K=64, N=72, r=5, dev="cuda", dtype=torch.bfloat16)
    batch = AdapterBatch([2, 0, 1], [4, 3, 2], 3)
    want = adapter_linear(x, w, a, b, batch, 1.5)
    whole = torch.cat((x.new_zeros(3), a.flatten(), b.flatten()))
    oa, ob = whole[3:3 + a.numel()].view(a.shape), whole[3 + a.numel():].view(b.shape)
    assert oa.data_ptr() % 16 and ob.data_ptr() % 16
    turned = a.transpose(2, 3).contiguous().transpose(2, 3)
    for p, q in ((oa, b), (a, ob), (oa, ob), (turned, b)):
        assert torch.equal(adapter_linear(x, w, p, q, batch, 1.5), want)
    p, q = oa.detach().requires_grad_(True), ob.detach().requires_grad_(True)
    y = adapter_linear(x, w, p, q, batch, 1.5)
    assert torch.equal(y.detach(), want)
    assert [g.shape for g in torch.autograd.grad(y, (p, q), torch.ones_like(y))] == [a.shape, b.shape]


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS, ids=range(len(LAYOUTS)))
def test_a_request_alone_answers_as_among_others(layout):
    """Up to the order of fp32 sums: how a reduction is split depends on the batch's size. Each way is within one
    rounding of y and one of each t of the formula."""
    from test_adapters import BF, formula

    ids, lengths, G, H, K, N, r, shared = layout
    gen = torch.Generator().manual_seed(6)
    rn = lambda *s: torch.randn(*s, generator=gen).to("cuda", torch.bfloat16)  # noqa: E731
    M = sum(lengths)
    x, w = (rn(M, K) if shared else rn(M, H, K)), rn(H, K, N) * 0.1
    a, b, scale = rn(G, H, r, K) * K ** -0.5, rn(G, H, r, N) * 0.2, torch.ones(G, device="cuda")
    batch = AdapterBatch(ids, lengths, G)
    y = adapter_linear(x, w, a, b, batch, scale)
    want, low, size, _ = formula(x, w, a, b, batch.adapter_of_row(), scale)
    bound = 2 * (BF * 1.01 * (want.abs() + low) + (K + 64) * 2.0 ** -23 * size)
    at = 0
    for g, n in zip(ids, lengths):
        rows = slice(at, at + n)
        alone = adapter_linear(x[rows], w, a, b, AdapterBatch([g], [n], G), scale)
        assert ((alone.double() - y[rows].double()).abs() <= bound[rows]).all()
        at += n
