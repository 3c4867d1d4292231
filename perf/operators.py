"""Cases of the operators for many adapters on one frozen model: ``adapter_linear`` (low-rank
adapters of many requests beside a shared projection), ``sample_tokens`` (temperature, top-k,
top-p and min-p with each request's own settings) and ``AdamWMany`` (one AdamW step over many
tensors, states in 32 or 8 bits). ``run`` computes them plainly in 32 bits, or with the
framework's kernels where ``own`` is true.

Sizes are the BDH-GPU projections (4 heads, 256 -> 8192 per head, decoder 32768 -> 256, adapter
rank 16), the tiny configuration's (4 heads, 64 -> 512), byte and subword vocabularies.
"""

import math

import torch

own = False

BLOCK = 256  # values that share one scale of an 8-bit state
ONE = 2.0 ** 40  # fixed-point one of a sampling weight
BETAS, EPS, DECAY, LR = (0.9, 0.999), 1e-8, 0.1, 1e-3


def listed():
    def adapter(name, rows, requests, adapters, H, K, N, rank, shared=True, train=False):
        return dict(name=name, op="adapter", rows=rows, requests=requests, adapters=adapters, H=H, K=K, N=N,
                    rank=rank, shared=shared, train=train)

    return [
        # one request's next token on the tiny configuration: latency
        adapter("adapter_token_tiny", 1, 1, 4, 4, 64, 512, 8),
        # one decode step of 48 requests, nearly each with an adapter of its own: the encoder
        adapter("adapter_tokens_encoder", 48, 48, 64, 4, 256, 8192, 16),
        # the same step's decoder projection, a long reduction, adapters shared by some requests
        adapter("adapter_tokens_decoder", 64, 64, 24, 1, 32768, 256, 16),
        # nine prompts of ragged lengths in one prefill batch: encoder, then decoder
        adapter("adapter_prompts_encoder", 4099, 9, 6, 4, 256, 8192, 16),
        adapter("adapter_prompts_decoder", 2500, 7, 7, 1, 32768, 256, 16),
        # a training batch of eight adapters, forward and backward
        adapter("adapter_train_encoder", 2048, 8, 8, 4, 256, 8192, 16, train=True),
        # sixteen byte-level requests
        dict(name="sample_bytes", op="sample", rows=16, vocab=256, half=False),
        # a few requests on a subword vocabulary, bf16 logits
        dict(name="sample_few", op="sample", rows=3, vocab=50000, half=True),
        # a full serving batch on a large vocabulary
        dict(name="sample_batch", op="sample", rows=200, vocab=128000, half=False),
        # small odd tensors (biases, gains, gates): latency
        dict(name="adamw_small_32bit", op="adamw", kind="odd", tensors=40, size=1500, bits=32, half=False),
        # sixteen adapters of the BDH-GPU model, bf16 gradients and working copies, 8-bit states
        dict(name="adamw_adapters_8bit", op="adamw", kind="adapters", tensors=96, size=0, bits=8, half=True),
        # the three shared projections of the whole model, 32-bit states
        dict(name="adamw_model_32bit", op="adamw", kind="even", tensors=3, size=8388608, bits=32, half=False),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(("adapter", "adapter", "sample", "adamw"))
    if op == "adapter":
        shape = rng.choice(("encoder", "decoder", "square"))
        if shape == "encoder":
            H, K, N = rng.choice((1, 2, 4)), 8 * log(8, 64), 8 * log(64, 1024)
        elif shape == "decoder":
            H, K, N = 1, 8 * log(256, 4096), 8 * log(8, 64)
        else:
            H, K, N = 1, 8 * log(16, 256), 8 * log(16, 256)
        most = min(4096, int(2.0e10 / (H * K * N)))
        requests = log(1, 64)
        rows = requests if rng.random() < 0.4 else max(requests, log(16, max(17, most)))
        return dict(op="adapter", rows=rows, requests=requests, adapters=log(1, 64), H=H, K=K, N=N,
                    rank=rng.choice((4, 5, 8, 16, 16, 24, 32, 64)), shared=H > 1 and rng.random() < 0.6,
                    train=rng.random() < 0.35)
    if op == "sample":
        vocab = log(250, 130000)
        return dict(op="sample", rows=log(1, max(2, min(256, 25000000 // vocab))), vocab=vocab,
                    half=rng.random() < 0.4)
    kind = rng.choice(("odd", "even"))
    tensors = log(1, 400)
    return dict(op="adamw", kind=kind, tensors=tensors, size=log(40, 24000000 // tensors), bits=rng.choice((8, 32)),
                half=rng.random() < 0.5)


# ------------------------------------------------------------------------------ inputs


def _generator(seed, device):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def _layout(case, seed):
    """The adapter of every row: ragged requests, adapters in random order, every ninth request without one."""
    g = torch.Generator().manual_seed(seed)
    R, M, G = case["requests"], case["rows"], case["adapters"]
    cuts = torch.randperm(M - 1, generator=g)[:R - 1].sort().values + 1 if R > 1 else torch.zeros(0, dtype=torch.long)
    edges = torch.cat((torch.zeros(1, dtype=torch.long), cuts, torch.full((1,), M)))
    order = torch.randperm(G, generator=g)
    ids = order[torch.arange(R) % G]
    ids[torch.arange(R) % 9 == 8] = -1
    return ids.tolist(), edges.diff().tolist()


def _adapter_inputs(case, seed):
    dev = torch.device("cuda")
    g = _generator(seed, dev)
    M, H, K, N, G, r = (case[k] for k in ("rows", "H", "K", "N", "adapters", "rank"))
    rn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x = rn(M, K) if H == 1 or case["shared"] else rn(M, H, K)
    if H == 1 and K > N:  # the decoder reads products of two rectified projections: sparse, not negative
        x = torch.relu(x) * torch.relu(rn(M, K))
    s = dict(x=x.bfloat16(), w=(rn(H, K, N) * 0.02).bfloat16(),
             a=((torch.rand(G, H, r, K, generator=g, device=dev) * 2 - 1) / math.sqrt(K)).bfloat16(),
             b=(rn(G, H, r, N) * 0.02).bfloat16(),
             scale=(torch.rand(G, generator=g, device=dev) + 0.5) * 16 / math.sqrt(r))
    if H == 1:
        s["w"], s["a"], s["b"] = s["w"][0], s["a"][:, 0], s["b"][:, 0]
    s["ids"], s["lengths"] = _layout(case, seed)
    if case["train"]:
        s["dy"] = (rn(M, N) if H == 1 else rn(M, H, N)).bfloat16()
        for k in ("x", "a", "b"):
            s[k].requires_grad_(True)
    return s


def _sample_inputs(case, seed):
    dev = torch.device("cuda")
    g = _generator(seed, dev)
    B, V = case["rows"], case["vocab"]
    rand = lambda: torch.rand(B, generator=g, device=dev)  # noqa: E731
    logits = torch.randn(B, V, generator=g, device=dev) * (1.0 + 3.0 * rand())[:, None]
    logits[:, : V // 50] = float("-inf")  # ids that are never answered
    pick = torch.rand(B, 4, generator=g, device=dev)
    temperature = torch.where(pick[:, 0] < 0.1, 0.0, 0.5 + rand())
    top_k = torch.where(pick[:, 1] < 0.5, 0, (1 + 200 * rand()).int()).int()
    top_p = torch.where(pick[:, 2] < 0.3, 1.0, 0.6 + 0.39 * rand())
    min_p = torch.where(pick[:, 3] < 0.6, 0.0, 0.1 * rand())
    return dict(logits=logits.bfloat16() if case["half"] else logits, u=rand(), temperature=temperature,
                top_k=top_k, top_p=top_p, min_p=min_p)


def _sizes(case):
    n = case["tensors"]
    if case["kind"] == "adapters":  # encoder a, b; encoder_v a, b; decoder a, b; rank 16
        return [16384, 524288, 16384, 524288, 524288, 4096] * (n // 6)
    if case["kind"] == "odd":  # from one value to twice the size, at odd places
        return [1 + (2 * case["size"] * ((7 * i) % n)) // n for i in range(n)]
    return [case["size"] - case["size"] % 8 + 8] * n


def _adamw_inputs(case, seed):
    dev = torch.device("cuda")
    g = _generator(seed, dev)
    sizes = _sizes(case)
    total = sum(sizes)
    flat = torch.randn(total, generator=g, device=dev) * 0.02
    shadow = flat.bfloat16() if case["half"] else None
    grad = torch.randn(total, generator=g, device=dev) * 1e-3 * torch.rand(total, generator=g, device=dev)
    grad = grad.bfloat16() if case["half"] else grad
    padded = sum(-(-n // BLOCK) * BLOCK for n in sizes)
    m = torch.randn(padded, generator=g, device=dev) * 2e-4
    v = torch.rand(padded, generator=g, device=dev).pow(4) * 1e-6
    valid = torch.cat([torch.arange(-(-n // BLOCK) * BLOCK) < n for n in sizes]).to(dev)
    m, v = m * valid, v * valid
    s = dict(sizes=sizes, flat=flat, shadow=shadow, params=list(flat.split(sizes)), grads=list(grad.split(sizes)),
             shadows=None if shadow is None else list(shadow.split(sizes)), t=10, seed=seed & 0xFFFF)
    if case["bits"] == 8:
        bits = _hash(padded, s["seed"], 10, dev)
        s["m"], s["m_scale"] = _encode(m, bits & 0xFFFF, False)
        s["v"], s["v_scale"] = _encode(v, bits >> 16, True)
    else:
        s["m"], s["v"] = m, v
    return s


def prepare(case, seed):
    s = {"adapter": _adapter_inputs, "sample": _sample_inputs, "adamw": _adamw_inputs}[case["op"]](case, seed)
    s["case"] = case
    if case["op"] == "adapter":
        ids = torch.repeat_interleave(torch.tensor(s["ids"]), torch.tensor(s["lengths"]))
        s["of_row"] = ids.to(s["x"].device)
    if own:  # the plan of a batch and the optimizer: what a program keeps from call to call
        if case["op"] == "adapter":
            from burn_dragon_b200.ops.adapters import AdapterBatch

            s["batch"] = AdapterBatch(s["ids"], s["lengths"], case["adapters"], device=s["x"].device)
        if case["op"] == "adamw":
            from burn_dragon_b200.train.optim import AdamWMany

            s["opt"] = AdamWMany(s["params"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
                                 state_bits=case["bits"], shadows=s["shadows"], seed=s["seed"])
            names = ("m", "v", "m_scale", "v_scale") if case["bits"] == 8 else ("m", "v")
            s["opt"].load_state_dict({"t": s["t"], **{k: s[k] for k in names}})
    return s


# ------------------------------------------------------------------------------ plain forms


def _adapter_plain(s):
    """Every row against every adapter, the others' columns set to zero: three products, no gather."""
    heads = s["w"].dim() == 3
    x, w, a, b = (s[k].detach().float() for k in ("x", "w", "a", "b"))
    if not heads:
        w, a, b = w[None], a[:, None], b[:, None]
    G, H, r, K = a.shape
    M, N = x.shape[0], w.shape[2]
    xs = x[:, None].expand(M, H, K) if x.dim() == 2 else x
    mask = (s["of_row"][:, None] == torch.arange(G, device=x.device)).float() * s["scale"]  # [M, G]
    mask = mask[:, :, None].expand(M, G, r).reshape(M, G * r)[:, None]  # [M, 1, G r]
    ah, bh = a.transpose(0, 1).reshape(H, G * r, K), b.transpose(0, 1).reshape(H, G * r, N)
    xh = xs.transpose(0, 1)  # [H, M, K]
    t = (xh @ ah.transpose(1, 2)) * mask.transpose(0, 1)  # [H, M, G r], scaled
    y = (xh @ w + t @ bh).transpose(0, 1)
    out = {"y": (y if heads else y[:, 0]).bfloat16().contiguous()}
    if s["case"]["train"]:
        dy = s["dy"].float()
        dyh = (dy if heads else dy[:, None]).transpose(0, 1)
        u = (dyh @ bh.transpose(1, 2)) * mask.transpose(0, 1)
        dx = dyh @ w.transpose(1, 2) + u @ ah
        dx = dx.sum(0) if x.dim() == 2 else dx.transpose(0, 1)
        da = (u.transpose(1, 2) @ xh).view(H, G, r, K).transpose(0, 1)
        db = (t.transpose(1, 2) @ dyh).view(H, G, r, N).transpose(0, 1)
        out |= {"dx": dx.bfloat16().contiguous(), "da": (da if heads else da[:, 0]).bfloat16().contiguous(),
                "db": (db if heads else db[:, 0]).bfloat16().contiguous()}
    return out


def _adapter_own(s):
    from burn_dragon_b200.ops.adapters import adapter_linear

    y = adapter_linear(s["x"], s["w"], s["a"], s["b"], s["batch"], s["scale"])
    if not s["case"]["train"]:
        return {"y": y}
    dx, da, db = torch.autograd.grad(y, (s["x"], s["a"], s["b"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "da": da, "db": db}


def _sample_plain(s):
    l = s["logits"].float()
    B, V = l.shape
    l = torch.where(l.isnan(), float("-inf"), l)
    top = l.amax(1, keepdim=True)
    t = s["temperature"][:, None]
    z = torch.where(l == top, 0.0, (l - top) * (1.0 / t))
    w = torch.where(l == float("-inf"), 0.0, torch.exp(z))
    W = (w * ONE).to(torch.int64)
    order = l.sort(dim=1, descending=True, stable=True).indices
    Ws = W.gather(1, order)
    k = torch.where(s["top_k"] > 0, s["top_k"], V)[:, None]
    keep = torch.arange(V, device=l.device)[None] < k
    Ws = torch.where(keep, Ws, 0)
    total = Ws.sum(1, keepdim=True)
    p = s["top_p"][:, None]
    reach = torch.ceil(total.double() * p.double()).to(torch.int64).clamp_min(1)
    reach = torch.where(p >= 1.0, total, reach)
    keep &= Ws.cumsum(1) - Ws < reach
    keep &= w.gather(1, order) >= s["min_p"][:, None].clamp_max(1.0)
    kept = torch.zeros_like(W).scatter_(1, order, torch.where(keep, Ws, 0))
    total = kept.sum(1)
    target = (s["u"].double() * total.double()).to(torch.int64).minimum(total - 1)
    token = (kept.cumsum(1) <= target[:, None]).sum(1)
    first = (l == top).to(torch.int8).argmax(1)
    greedy = ~(s["temperature"] > 0)
    token = torch.where(greedy, first, token.clamp_max(V - 1))
    logprob = z.gather(1, token[:, None])[:, 0] - (total.float() * (1.0 / ONE)).log()
    logprob = torch.where(greedy, 0.0, logprob)
    empty = top[:, 0] == float("-inf")
    return {"tokens": torch.where(empty, -1, token), "logprobs": torch.where(empty, float("-inf"), logprob)}


def _sample_own(s):
    from burn_dragon_b200.ops.sampling import sample_tokens

    tokens, logprobs = sample_tokens(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    return {"tokens": tokens, "logprobs": logprobs}


def _hash(n, seed, t, device):
    """32 bits for each of n indexes from the seed and the step, as int64."""
    low = 0xFFFFFFFF
    key = (seed * 0x9E3779B1 + t * 0x85EBCA77) & low
    h = (torch.arange(n, device=device) * 0x9E3779B1 + key) & low
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & low
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & low
    return h ^ (h >> 16)


def _decode(code, scale):
    return (code.float().view(-1, BLOCK) * scale[:, None]).reshape(-1)


def _encode(x, bits16, floor):
    """e4m3 values and one scale for each block: absmax / 256; a value between two codes takes the upper one where
    its 16 random bits carry. With `floor`, what is above zero keeps the lowest code at least."""
    blocks = x.view(-1, BLOCK)
    amax = blocks.abs().amax(1, keepdim=True)
    fine = (amax >= 2.0 ** -110) & (amax < float("inf"))
    inverse = torch.where(fine, 256.0 / amax, 0.0)
    scale = torch.where(fine, amax * 2.0 ** -8, torch.where(amax < 2.0 ** -110, 0.0, amax))
    y = (blocks.abs() * inverse) * 2.0 ** -120
    code = (y.view(torch.int32) + (bits16.view(-1, BLOCK) << 4).to(torch.int32)) >> 20
    if floor:
        code = torch.where(blocks > 0, code.clamp_min(1), code)
    code = torch.where(blocks < 0, code + 128, code) * fine
    return code.to(torch.uint8).view(torch.float8_e4m3fn).reshape(-1), scale[:, 0]


def _adamw_plain(s):
    s["t"] += 1
    sizes, bits = s["sizes"], s["case"]["bits"]
    pad = lambda ts: torch.cat([torch.nn.functional.pad(x.float(), (0, -x.numel() % BLOCK)) for x in ts])  # noqa: E731
    g, p = pad(s["grads"]), pad(s["params"])
    m = _decode(s["m"], s["m_scale"]) if bits == 8 else s["m"]
    v = _decode(s["v"], s["v_scale"]) if bits == 8 else s["v"]
    (b1, b2), t = BETAS, s["t"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    p = p * (1 - LR * DECAY) - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS)
    parts = p.split([-(-n // BLOCK) * BLOCK for n in sizes])
    s["flat"].copy_(torch.cat([q[:n] for q, n in zip(parts, sizes)]))
    if s["shadow"] is not None:
        s["shadow"].copy_(s["flat"])
    if bits == 8:
        h = _hash(m.numel(), s["seed"], t, m.device)
        (m, m_scale), (v, v_scale) = _encode(m, h & 0xFFFF, False), _encode(v, h >> 16, True)
        s["m_scale"].copy_(m_scale)
        s["v_scale"].copy_(v_scale)
    s["m"].copy_(m)
    s["v"].copy_(v)
    return _adamw_out(s, s)


def _adamw_out(s, state):
    names = ("m", "v", "m_scale", "v_scale") if s["case"]["bits"] == 8 else ("m", "v")
    out = {"params": s["flat"], **{k: state[k] for k in names}}
    return out if s["shadow"] is None else {**out, "shadow": s["shadow"]}


def _adamw_own(s):
    s["opt"].step(s["grads"])
    return _adamw_out(s, s["opt"].state)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"adapter": _adapter_own, "sample": _sample_own, "adamw": _adamw_own}[op](state)
    return {"adapter": _adapter_plain, "sample": _sample_plain, "adamw": _adamw_plain}[op](state)


# ------------------------------------------------------------------------------ what a pass cannot do without


def work(case):
    if case["op"] == "adapter":
        M, H, K, N, r = (case[k] for k in ("rows", "H", "K", "N", "rank"))
        R = case["requests"]
        used = len({i % case["adapters"] for i in range(R) if i % 9 != 8})
        some = M * (R - R // 9) // R  # rows with an adapter
        x = M * (K if H == 1 or case["shared"] else H * K)
        weights, adapters, y = H * K * N, H * r * (K + N), M * H * N
        base, low = 2 * M * H * K * N, 2 * some * H * r * (K + N)
        if not case["train"]:
            return {"bytes": 2 * (x + weights + used * adapters + y), "flops": base + low}
        # y, then dx, da, db: x, w and dy once more, every adapter's gradient written
        return {"bytes": 2 * (2 * x + weights + used * adapters + 2 * y + case["adapters"] * adapters),
                "flops": 2 * base + 3 * low}
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["half"] else 4) + case["rows"] * 32, "flops": 4 * n}
    n = sum(_sizes(case))
    state = 2 * (1 + 4 / BLOCK) * 2 if case["bits"] == 8 else 16
    return {"bytes": n * (8 + (4 if case["half"] else 4) + state), "flops": 14 * n}


# ------------------------------------------------------------------------------ the definition, in 64 bits


def exact(case, seed):
    if case["op"] == "adapter":
        return _adapter_exact(_adapter_inputs(case, seed), case)
    if case["op"] == "sample":
        return _sample_exact(_sample_inputs(case, seed), case)
    return _adamw_exact(_adamw_inputs(case, seed), case)


def _adapter_exact(s, case):
    """Request by request, each with its own adapter's weights added to the projection."""
    x, w, a, b, scale = (s[k].detach().double() for k in ("x", "w", "a", "b", "scale"))
    heads = w.dim() == 3
    if not heads:
        w, a, b = w[None], a[:, None], b[:, None]
    H, shared = w.shape[0], x.dim() == 2
    dy = None
    if case["train"]:
        dy = s["dy"].double() if heads else s["dy"].double()[:, None]
    y = x.new_zeros(case["rows"], H, w.shape[2])
    dx = x.new_zeros(case["rows"], H, w.shape[1])
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    at = 0
    for g, n in zip(s["ids"], s["lengths"]):
        rows = slice(at, at + n)
        for h in range(H):
            xr = x[rows] if shared else x[rows, h]
            full = w[h] if g < 0 else w[h] + scale[g] * a[g, h].T @ b[g, h]
            y[rows, h] = xr @ full
            if dy is not None:
                dx[rows, h] = dy[rows, h] @ full.T
                if g >= 0:
                    outer = scale[g] * (xr.T @ dy[rows, h])
                    da[g, h] += b[g, h] @ outer.T
                    db[g, h] += a[g, h] @ outer
        at += n
    out = {"y": y if heads else y[:, 0]}
    if dy is not None:
        out |= {"dx": dx.sum(1) if shared else dx, "da": da if heads else da[:, 0], "db": db if heads else db[:, 0]}
    return out


def _sample_exact(s, case):
    """The log-probabilities, row by row; a token is a whole number and has no value in 64 bits."""
    logits, V = s["logits"].double().cpu(), case["vocab"]
    settings = zip(*(s[k].double().tolist() for k in ("u", "temperature", "top_k", "top_p", "min_p")))
    found = []
    for row, (u, t, k, p, low) in zip(logits, settings):
        if t <= 0:
            found.append(0.0)
            continue
        prob = torch.softmax(row / t, 0)
        ordered, index = prob.sort(descending=True, stable=True)
        n = int(k) if 0 < k < V else V
        share = ordered[:n] / ordered[:n].sum()
        if p < 1.0:
            n = max(1, int((share.cumsum(0) - share < p).sum()))
        n = max(1, min(n, int((ordered >= low * ordered[0]).sum())))
        kept = torch.zeros_like(prob)
        kept[index[:n]] = ordered[:n] / ordered[:n].sum()
        token = min(int((kept.cumsum(0) <= u).sum()), V - 1)
        found.append(float(kept[token].log()))
    return {"tokens": None, "logprobs": torch.tensor(found, dtype=torch.float64)}


def _adamw_exact(s, case):
    """Tensor by tensor with every value in 64 bits; states of 8 bits are rounded by the same random bits."""
    t, (b1, b2), eight = s["t"] + 1, BETAS, case["bits"] == 8
    bits = _hash(s["m"].numel(), s["seed"], t, s["m"].device)
    params, ms, vs, m_scales, v_scales = [], [], [], [], []
    at = 0
    for p, g, n in zip(s["params"], s["grads"], s["sizes"]):
        size = -(-n // BLOCK) * BLOCK
        m, v = s["m"][at:at + size].double(), s["v"][at:at + size].double()
        if eight:
            blocks = slice(at // BLOCK, (at + size) // BLOCK)
            m = m * s["m_scale"][blocks].double().repeat_interleave(BLOCK)
            v = v * s["v_scale"][blocks].double().repeat_interleave(BLOCK)
        g = torch.cat((g.double(), g.new_zeros(size - n).double()))
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        step = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS)
        params.append(p.double() * (1 - LR * DECAY) - LR * step[:n])
        if eight:
            h = bits[at:at + size]
            (m, m_scale), (v, v_scale) = _round8(m, h & 0xFFFF, False), _round8(v, h >> 16, True)
            m_scales.append(m_scale)
            v_scales.append(v_scale)
        ms.append(m)
        vs.append(v)
        at += size
    out = {"params": torch.cat(params), "m": torch.cat(ms), "v": torch.cat(vs)}
    if eight:
        out |= {"m_scale": torch.cat(m_scales), "v_scale": torch.cat(v_scales)}
    return {**out, "shadow": torch.cat(params)} if case["half"] else out


def _round8(x, bits16, floor):
    """Values on the e4m3 grid of their block, rounded up where the random fraction reaches what is above the grid."""
    blocks = x.view(-1, BLOCK)
    scale = blocks.abs().amax(1) / 256
    unit = torch.where(scale[:, None] > 0, blocks.abs() / scale[:, None], 0.0)
    exponent = torch.floor(torch.log2(unit.clamp_min(2.0 ** -6)))
    grid = torch.exp2(exponent - 3)
    up = bits16.view(-1, BLOCK).double() / 65536
    value = torch.floor(unit / grid + up) * grid
    if floor:
        value = torch.where(blocks > 0, value.clamp_min(2.0 ** -9), value)
    return (value * blocks.sign()).reshape(-1), scale
