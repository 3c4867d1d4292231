"""Next-token sampling with each request's own settings (``csrc/sampling.cu``).

``sample_tokens`` draws one token per row of logits from given uniform numbers, so a run can be
repeated, and returns its log-probability under the distribution it was drawn from (the behaviour
policy's, which policy-gradient objectives divide by): a constant, without a graph. The policy's own
log-probability, with its gradient, is computed from the logits. In the order "value descending, index ascending":

1. ``temperature`` T: weights exp((l - max) / T); T <= 0 answers the first maximum, log-probability 0, and +inf
   counts as the largest fp32 number (every token that is not masked by -inf is as likely as another);
2. ``top_k`` k > 0: the first k;
3. ``top_p`` p < 1: of those, the shortest prefix whose share reaches p (the first token at least);
4. ``min_p``: those whose weight is at least min_p times the largest;
5. the token is the first (in index order) whose running share of what is left exceeds ``u``.

Ties go to the lowest index. A NaN logit is never drawn; a row without a finite or +inf logit answers
token -1 with log-probability -inf. Weights are summed as whole numbers of 2^-40, so a
row's token does not depend on the batch it is in.
"""

from __future__ import annotations

import torch

from .. import _ext

MAX_VOCAB = 262144
_ONE = 2.0 ** 40


def _setting(value, rows: int, device, dtype, what: str):
    """A per-row tensor (or None) and the number that stands in for it."""
    if isinstance(value, torch.Tensor):
        if value.shape != (rows,):
            raise ValueError(f"{what} must be a number or one value per row, got shape {tuple(value.shape)}")
        if value.device != device or value.dtype != dtype:
            value = value.to(device, dtype)
        return value.contiguous(), 0
    return None, value


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0) -> tuple[torch.Tensor, torch.Tensor]:
    """logits [B, V] (fp32 or bf16 on CUDA; V <= 262144), u [B] uniform in [0, 1); a setting is a number
    for all rows or a tensor [B]. Returns (tokens [B] int64, logprobs [B] fp32)."""
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be [rows, vocabulary], got shape {tuple(logits.shape)}")
    B, V = logits.shape
    dev = logits.device
    if not isinstance(u, torch.Tensor):
        raise ValueError("u must be a tensor of one uniform number per row")
    u, _ = _setting(u, B, dev, torch.float32, "u")
    f32 = torch.float32
    t, t0 = _setting(temperature, B, dev, f32, "temperature")
    k, k0 = _setting(top_k, B, dev, torch.int32, "top_k")
    p, p0 = _setting(top_p, B, dev, f32, "top_p")
    m, m0 = _setting(min_p, B, dev, f32, "min_p")
    k0 = 0 if k0 is None else int(k0)
    if not logits.is_cuda:
        full = lambda x, x0, dt: torch.full((B,), x0, dtype=dt) if x is None else x  # noqa: E731
        with torch.no_grad():  # whole-number sums have no derivative: a graph would lack the normaliser's part
            return sample_tokens_ref(logits, u, full(t, t0, f32), full(k, k0, torch.int32), full(p, p0, f32),
                                     full(m, m0, f32))
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"sample_tokens takes fp32 or bf16 logits, not {logits.dtype}")
    if V > MAX_VOCAB:
        raise ValueError(f"sample_tokens takes a vocabulary of up to {MAX_VOCAB} tokens, not {V}")
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    tokens = torch.empty(B, dtype=torch.long, device=dev)
    logprobs = torch.empty(B, dtype=f32, device=dev)
    _ext.load().sample_tokens(logits, u, t, t0, k, k0, p, p0, m, m0, tokens, logprobs)
    return tokens, logprobs


def sample_tokens_ref(logits, u, temperature, top_k, top_p, min_p):
    """The same rule with a sort, in elementary operations (the CPU path)."""
    l = logits.float()
    B, V = l.shape
    l = torch.where(l.isnan(), float("-inf"), l)
    top = l.amax(1, keepdim=True)
    z = torch.where(l == top, 0.0, (l - top) * (1.0 / temperature[:, None].clamp_max(torch.finfo(torch.float32).max)))
    w = torch.where(l == float("-inf"), 0.0, z.exp())
    W = (w * _ONE).to(torch.int64)
    order = l.sort(dim=1, descending=True, stable=True).indices
    Ws = W.gather(1, order)
    k = torch.where(top_k > 0, top_k, V)[:, None]
    keep = torch.arange(V, device=l.device)[None] < k
    Ws = Ws * keep
    total = Ws.sum(1, keepdim=True)
    p = top_p[:, None]
    reach = torch.ceil(total.double() * p.double()).to(torch.int64).clamp_min(1)
    keep &= Ws.cumsum(1) - Ws < torch.where(p >= 1.0, total, reach)
    keep &= w.gather(1, order) >= min_p[:, None].clamp_max(1.0)
    kept = torch.zeros_like(W).scatter_(1, order, Ws * keep)
    total = kept.sum(1)
    target = (u.double() * total.double()).to(torch.int64).minimum(total - 1)
    token = (kept.cumsum(1) <= target[:, None]).sum(1).clamp_max(V - 1)
    logprob = z.gather(1, token[:, None])[:, 0] - (total.float() / _ONE).log()
    greedy, empty = ~(temperature > 0), top[:, 0] == float("-inf")
    token = torch.where(greedy, (l == top).to(torch.int8).argmax(1), token)
    logprob = torch.where(greedy, 0.0, logprob)
    return torch.where(empty, -1, token), torch.where(empty, float("-inf"), logprob)
