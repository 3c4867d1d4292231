"""sample_tokens at the ends of its settings, and rows that are hard for the paths of long vocabularies."""

import pytest
import torch
from test_sampling import hard_rows

from burn_dragon_b200.ops.sampling import sample_tokens, sample_tokens_ref

INF = float("inf")
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def same(got, want, names):
    for b, name in enumerate(names):
        assert int(got[0][b]) == int(want[0][b]), name
        assert torch.allclose(got[1][b], want[1][b], rtol=1e-6, atol=2e-6), name


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("V", [64, 1030, 5003, 33000])  # the last three end inside a vector of four
@pytest.mark.parametrize("k,p,low", [(0, 1.0, 0.0), (0, 0.5, 0.0), (7, 1.0, 0.0), (7, 0.5, 0.0), (0, 0.9, 1.0)])
def test_an_infinite_temperature_draws_evenly_from_what_is_not_masked(V, k, p, low, dev):
    logits = torch.randn(3, V, generator=torch.Generator().manual_seed(V))
    logits[1, ::2] = -INF
    logits[2] = -INF
    logits[2, V - 1] = 1.0
    u = torch.tensor([0.3, 0.7, 0.5])
    tokens, logprobs = sample_tokens(logits.to(dev), u.to(dev), INF, k, p, low)
    for b in range(3):
        order = logits[b].sort(descending=True, stable=True).indices
        order = order[:int((logits[b] > -INF).sum())]  # weights of one, all of them
        n = min(k, len(order)) if k else len(order)
        n = -int(-n * torch.tensor(p, dtype=torch.float32).double() // 1) if p < 1.0 else n
        kept = order[:n].sort().values
        assert int(tokens[b]) == int(kept[int(float(u[b]) * n)])
        assert abs(float(logprobs[b]) + torch.tensor(float(n)).log()) < 1e-5


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("k,p", [(0, 1.0), (0, 0.6), (5, 1.0)])
def test_an_infinite_logit_at_an_infinite_temperature(k, p, dev):
    logits = torch.linspace(-1, 1, 2050)
    logits[[700, 1500]] = INF
    tokens, logprobs = sample_tokens(logits.expand(2, -1).contiguous().to(dev), torch.tensor([0.2, 0.9]).to(dev), INF, k, p)
    assert tokens.tolist() == [700, 1500]
    assert torch.allclose(logprobs.cpu(), torch.full((2,), 0.5).log(), atol=1e-6)


@pytest.mark.parametrize("dev", DEVICES)
def test_log_probabilities_are_constants_on_every_device(dev):
    logits = torch.randn(3, 50, device=dev, requires_grad=True)
    temperature = torch.ones(3, device=dev, requires_grad=True)
    tokens, logprobs = sample_tokens(logits, torch.rand(3, device=dev), temperature, 5, 0.9)
    assert not logprobs.requires_grad and not tokens.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("V", [64, 5000, 33000])
@pytest.mark.parametrize("k,p,low", [(0, 1.0, 0.0), (0, 0.3, 0.0), (40, 0.6, 0.0), (0, 0.9, 0.5)])
def test_hard_rows_at_an_infinite_temperature(V, k, p, low):
    names, logits = hard_rows(V)
    u = torch.rand(len(names), generator=torch.Generator().manual_seed(V))
    full = [torch.full((len(names),), v, device="cuda") for v in (INF, k, p, low)]
    same(sample_tokens(logits.cuda(), u.cuda(), INF, k, p, low), sample_tokens_ref(logits.cuda(), u.cuda(), *full), names)


def long_rows(V):
    """hard_rows, and rows whose border lies among equal or nearly equal weights."""
    names, logits = hard_rows(V)
    more = {
        "two values": torch.arange(V).remainder(2).float() * 1e-6,
        "one heavy value": torch.zeros(V).index_fill(0, torch.tensor([V // 2]), 12.0),
        "a geometric fall": -torch.arange(V).float() * 1e-2,
        "equal but for the last bits": torch.full((V,), 2.0).add(torch.arange(V).remainder(3).float() * 2.0 ** -22),
        "a plateau below a few": torch.zeros(V).index_fill(0, torch.arange(0, V, 997), 3.0),
    }
    return names + list(more), torch.cat((logits, torch.stack(list(more.values()))))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [70001, 131073, 262144])  # slices of more than 8192 values: windows from a sample
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,k,p,low", [(1.0, 0, 0.3, 0.0), (0.7, 0, 0.95, 0.0), (1.0, 0, 0.0, 0.0), (1e-3, 0, 0.5, 0.0),
                                       (1e30, 0, 0.5, 0.0), (1.0, 300, 0.6, 0.0), (1.0, 2000, 1.0, 0.0), (1.0, 0, 0.9, 0.4),
                                       (INF, 0, 0.7, 0.0)])
def test_hard_rows_of_long_vocabularies(V, dtype, t, k, p, low):
    names, logits = long_rows(V)
    logits = logits.to(dtype).cuda()
    u = torch.rand(len(names), generator=torch.Generator().manual_seed(V)).cuda()
    full = [torch.full((len(names),), v, device="cuda") for v in (t, k, p, low)]
    same(sample_tokens(logits, u, t, k, p, low), sample_tokens_ref(logits, u, *full), names)
