"""Sampling with each request's own settings, against a sort in 64-bit and whole numbers."""

import math

import pytest
import torch

from burn_dragon_b200.ops.sampling import sample_tokens, sample_tokens_ref

F32 = torch.float32
LOW = torch.finfo(F32).min


def row_rule(l, u, t, k, p, low):
    """One row in Python: the kept tokens with their share, in index order (64 bits), and the token."""
    l = [float("-inf") if math.isnan(v) else v for v in l]
    top = max(l)
    if top == float("-inf"):
        return None, -1
    if not t > 0:
        return None, l.index(top)
    w = [1.0 if v == top else 0.0 if v == float("-inf") else math.exp(max((v - top) / t, -800.0)) for v in l]
    order = sorted(range(len(l)), key=lambda i: (-l[i], i))
    order = [i for i in order if w[i] >= 2.0 ** -40]  # a weight below 2^-40 is zero
    if 0 < k < len(l):
        order = order[:int(k)]
    if p < 1.0:
        whole, run, n = math.fsum(w[i] for i in order), 0.0, 0
        while n < len(order) and (n == 0 or run < p * whole):
            run += w[order[n]]
            n += 1
        order = order[:n]
    order = [i for i in order if w[i] >= min(low, 1.0)]
    whole = math.fsum(w[i] for i in order)
    kept = {i: w[i] / whole for i in sorted(order)}
    run = 0.0
    for i, share in kept.items():
        run += share
        if run > u:
            return kept, i
    return kept, i


def settings(B, gen, V):
    pick = torch.rand(B, 5, generator=gen)
    t = torch.where(pick[:, 0] < 0.15, 0.0, 0.3 + 1.5 * pick[:, 0])
    k = torch.where(pick[:, 1] < 0.4, 0, (1 + pick[:, 1] * min(V, 60)).int()).int()
    p = torch.where(pick[:, 2] < 0.3, 1.0, pick[:, 2])
    low = torch.where(pick[:, 3] < 0.5, 0.0, 0.3 * pick[:, 3])
    return torch.rand(B, generator=gen), t, k, p, low


def agree(got, logits, u, t, k, p, low):
    """The token of the sorted rule; another one only where u (or p) lies within rounding of a border."""
    tokens, logprobs = got[0].cpu(), got[1].cpu()
    for b in range(logits.shape[0]):
        row = logits[b].float().tolist()
        args = [float(v[b]) for v in (u, t, k, p, low)]
        kept, want = row_rule(row, *args)
        if kept is None:
            assert int(tokens[b]) == want
            assert float(logprobs[b]) == (float("-inf") if want < 0 else 0.0)
            continue
        token = int(tokens[b])
        if token != want:  # fp32 weights: allow what a change of u and p by 1e-6 allows
            near = set()
            for du in (-1e-6, 1e-6):
                for dp in (-1e-6, 0.0, 1e-6):
                    near.add(row_rule(row, args[0] + du, args[1], args[2], args[3] + dp, args[4])[1])
            assert token in near, (b, token, want)
        elif token in kept:
            # z and log in fp32: 2^-23 of their sizes, the weights' sum to 1e-6
            assert abs(float(logprobs[b]) - math.log(kept[token])) < 2e-6 * (10 + abs(math.log(kept[token])))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, torch.bfloat16])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 31), (16, 256), (7, 1000), (4, 2049), (2, 4097), (3, 50001), (2, 131073)])
def test_kernel_draws_the_sorted_rules_token(B, V, dtype):
    gen = torch.Generator().manual_seed(B * V)
    logits = (torch.randn(B, V, generator=gen) * 3).to(dtype)
    logits[:, V // 2:V // 2 + V // 20] = float("-inf")
    args = settings(B, gen, V)
    agree(sample_tokens(logits.cuda(), *(a.cuda() for a in args)), logits, *args)


@pytest.mark.gpu
def test_kernel_equals_the_elementary_operations():
    """Whole-number sums: the kernel and a sort of the same weights agree token for token."""
    gen = torch.Generator().manual_seed(5)
    for B, V in ((200, 256), (64, 5003), (9, 70000)):
        logits = (torch.randn(B, V, generator=gen) * 2).cuda()
        args = [a.cuda() for a in settings(B, gen, V)]
        got, want = sample_tokens(logits, *args), sample_tokens_ref(logits, *args)
        assert torch.equal(got[0], want[0])
        assert torch.allclose(got[1], want[1], rtol=1e-6, atol=2e-6)


def hard_rows(V):
    inf, nan = float("inf"), float("nan")
    rows = {
        "nothing left": torch.full((V,), -inf),
        "only NaN": torch.full((V,), nan),
        "one finite": torch.full((V,), -inf).index_fill(0, torch.tensor([V - 1]), -3.0),
        "lowest values": torch.full((V,), LOW),
        "masked by the lowest value": torch.cat((torch.full((V - V // 3,), LOW), torch.linspace(-1, 1, V // 3))),
        "all equal": torch.full((V,), 1.25),
        "plus infinity": torch.linspace(-1, 1, V).index_fill(0, torch.tensor([V // 3, V // 2]), inf),
        "NaN among values": torch.linspace(-2, 2, V).index_fill(0, torch.tensor([0, V - 1]), nan),
        "zeros of both signs": torch.zeros(V).index_fill(0, torch.arange(0, V, 2), -0.0),
        "ties at the border": torch.arange(V).remainder(4).float(),
        "one bucket": 1.0 + torch.linspace(0, 1e-3, V),
        "huge": torch.linspace(-3e38, 3e38, V),
    }
    return list(rows), torch.stack(list(rows.values()))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [64, 5000, 33000])
@pytest.mark.parametrize("t,k,p,low", [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.0, 0, 0.3, 0.0), (1.3, 40, 0.6, 0.01),
                                       (0.0, 3, 0.5, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0),
                                       (1e-30, 0, 0.9, 0.0), (5e-324, 0, 1.0, 0.0), (1e30, 0, 0.5, 0.5)])
def test_rows_where_it_can_go_wrong(V, t, k, p, low):
    names, logits = hard_rows(V)
    B = len(names)
    u = torch.rand(B, generator=torch.Generator().manual_seed(V))
    got = sample_tokens(logits.cuda(), u.cuda(), t, k, p, low)
    want = sample_tokens_ref(logits.cuda(), u.cuda(), *(torch.full((B,), v, device="cuda") for v in (t, k, p, low)))
    for b, name in enumerate(names):
        assert int(got[0][b]) == int(want[0][b]), name
        assert torch.allclose(got[1][b], want[1][b], rtol=1e-6, atol=2e-6), name
    assert int(got[0][0]) == -1 and int(got[0][1]) == -1 and int(got[0][2]) == V - 1
    assert int(got[0][6]) in (V // 3, V // 2)


@pytest.mark.gpu
def test_a_row_does_not_depend_on_its_batch():
    gen = torch.Generator().manual_seed(1)
    logits = torch.randn(180, 9000, generator=gen).cuda()
    args = [a.cuda() for a in settings(180, gen, 9000)]
    tokens, logprobs = sample_tokens(logits, *args)
    for b in (0, 77, 179):
        alone = sample_tokens(logits[b:b + 1], *(a[b:b + 1] for a in args))
        assert int(alone[0]) == int(tokens[b]) and float(alone[1]) == float(logprobs[b])


@pytest.mark.gpu
def test_strided_rows_ends_of_u_and_another_stream():
    gen = torch.Generator().manual_seed(2)
    wide = torch.randn(6, 777, generator=gen).cuda()
    part = wide[:, 5:705]  # rows that start at odd places
    u = torch.tensor([0.0, 0.1, 0.5, 0.9, 1.0 - 2.0 ** -24, 1.0], device="cuda")
    got = sample_tokens(part, u)
    want = sample_tokens(part.contiguous(), u)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert int(got[0][0]) == 0 and int(got[0][5]) == 699
    turned = part.t().contiguous().t()
    assert torch.equal(sample_tokens(turned, u)[0], want[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = sample_tokens(part, u)
    side.synchronize()
    assert torch.equal(again[0], want[0])
    assert sample_tokens(part[:0], u[:0])[0].numel() == 0


@pytest.mark.gpu
def test_shares_of_many_draws():
    """2^16 evenly spaced u: each token is drawn in proportion to its probability, to one draw."""
    logits = torch.tensor([0.3, -1.0, 2.0, 0.3, -5.0, 1.0], device="cuda")
    n = 1 << 16
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tokens, _ = sample_tokens(logits.expand(n, 6).contiguous(), u, 0.8)
    share = torch.bincount(tokens, minlength=6).double()
    want = torch.softmax(logits.double() / 0.8, 0) * n
    assert (share - want).abs().max() <= 1.1


def test_cpu_path_follows_the_rule():
    gen = torch.Generator().manual_seed(7)
    logits = torch.randn(40, 50, generator=gen) * 2
    args = settings(40, gen, 50)
    agree(sample_tokens(logits, *args), logits, *args)
    _, logits = hard_rows(64)
    u = torch.full((logits.shape[0],), 0.4)
    tokens, logprobs = sample_tokens(logits, u, 0.9, 7, 0.8, 0.0)
    assert tokens[:3].tolist() == [-1, -1, 63] and logprobs[0] == float("-inf")


def test_refusals():
    logits, u = torch.zeros(3, 8), torch.zeros(3)
    with pytest.raises(ValueError, match="rows, vocabulary"):
        sample_tokens(logits[0], u)
    with pytest.raises(ValueError, match="rows, vocabulary"):
        sample_tokens(logits[:, :0], u)
    with pytest.raises(ValueError, match="u must be"):
        sample_tokens(logits, u[:2])
    with pytest.raises(ValueError, match="u must be"):
        sample_tokens(logits, 0.5)
    with pytest.raises(ValueError, match="temperature"):
        sample_tokens(logits, u, torch.ones(2))
    with pytest.raises(ValueError, match="top_p"):
        sample_tokens(logits, u, 1.0, 0, torch.ones(3, 1))


@pytest.mark.gpu
def test_refusals_on_the_device():
    u = torch.zeros(1, device="cuda")
    with pytest.raises(TypeError, match="fp32 or bf16"):
        sample_tokens(torch.zeros(1, 8, device="cuda", dtype=torch.float64), u)
    with pytest.raises(ValueError, match="262144"):
        sample_tokens(torch.zeros(1, 262145, device="cuda"), u)
