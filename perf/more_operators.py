"""Cases of the feed-forward operators: ``linear_act`` (a matrix product with bias, activation and
residual in its epilogue), ``gated_linear`` (two projections, their activations and the product in one
kernel) and activations held in 8 bits (``pack_activation``, and ``keep="8bit"`` of the other two).
``run`` computes them plainly in 32 bits, or with the framework's kernels where ``own`` is true.

Sizes are the BDH-GPU projections (4 heads, 256 -> 8192 per head, decoder 32768 -> 256), the tiny
configuration's width, and feed-forward blocks of a few thousand columns.
"""

import math

import torch

own = False

BLOCK = 32  # values that share one scale of an 8-bit activation
LARGEST = 448.0  # the largest e4m3 value


def listed():
    def linear(name, rows, K, N, act="none", bias=False, residual=False, turned=False, half=False, train=False, keep=None):
        return dict(name=name, op="linear", rows=rows, K=K, N=N, act=act, bias=bias, residual=residual, turned=turned,
                    half=half, train=train, keep=keep)

    def gated(name, rows, H, K, N, act="relu", up="relu", z=True, half=False, train=False, keep=None):
        return dict(name=name, op="gated", rows=rows, H=H, K=K, N=N, act=act, up=up, z=z, half=half, train=train, keep=keep)

    return [
        # one token through the widening half of a small transformer block: latency
        linear("linear_token_tiny", 1, 64, 256, act="gelu", bias=True, turned=True),
        # one decode step of 48 requests: the decoder projection added to the stream, a long reduction
        linear("linear_tokens_decoder", 48, 32768, 256, residual=True),
        # prompts of ragged lengths through the widening half of a block, the weight laid out as torch.nn.Linear keeps it
        linear("linear_prompts", 4099, 1024, 4096, act="gelu", bias=True, turned=True),
        # a training batch, forward and backward
        linear("linear_train", 4096, 1024, 4096, act="gelu", bias=True, train=True, keep="16bit"),
        # odd sizes, fp16, pre-activations held in 8 bits
        linear("linear_train_ragged_8bit", 1777, 328, 1000, act="silu", bias=True, residual=True, half=True, train=True,
               keep="8bit"),
        # one token's gated step of the BDH-GPU layer, each head with its own second input
        gated("gated_token", 1, 4, 256, 8192),
        # a decode step of 64 requests
        gated("gated_tokens", 64, 4, 256, 8192),
        # prompts in one prefill batch
        gated("gated_prompts", 4099, 4, 256, 8192),
        # a training batch, the pre-activations computed again in the backward pass
        gated("gated_train", 4096, 4, 256, 8192, train=True, keep="recompute"),
        # a gated block with one input and one smooth activation, fp16, pre-activations held in 8 bits
        gated("gated_train_silu_8bit", 2500, 1, 1024, 2816, act="silu", up="none", z=False, half=True, train=True, keep="8bit"),
        # a small activation, held and read back: latency
        dict(name="act8_small", op="act8", rows=48, N=1000, type="fp32"),
        # one layer's pre-activations of the BDH-GPU model
        dict(name="act8_layer", op="act8", rows=4096, N=32768, type="bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))

    op = rng.choice(("linear", "linear", "gated", "gated", "act8"))
    if op == "act8":
        N = log(1, 33000)
        return dict(op="act8", rows=log(1, max(2, min(8000, 130000000 // N))), N=N, type=rng.choice(("bf16", "fp16", "fp32")))
    train = rng.random() < 0.5
    half = rng.random() < 0.4
    keep = rng.choice(("recompute", "16bit", "8bit")) if train else None
    if op == "linear":
        shape = rng.choice(("wide", "long", "square"))
        if shape == "wide":
            K, N = 8 * log(4, 128), 8 * log(64, 1024)
        elif shape == "long":
            K, N = 8 * log(256, 4096), 8 * log(8, 64)
        else:
            K, N = 8 * log(8, 400), 8 * log(8, 400)
        if rng.random() < 0.15:  # no multiples of anything
            K, N = K - rng.randrange(0, 8), N - rng.randrange(0, 8)
        most = max(16, min(4096, int((1.6e10 if train else 1.7e10) / (K * N))))
        rows = log(1, 64) if rng.random() < 0.4 else log(16, most)
        return dict(op="linear", rows=rows, K=K, N=N, act=rng.choice(("none", "relu", "silu", "gelu")),
                    bias=rng.random() < 0.6, residual=rng.random() < 0.4, turned=rng.random() < 0.5, half=half, train=train,
                    keep=keep)
    H = rng.choice((1, 1, 2, 4))
    K, N = 8 * log(8, 128), 8 * log(32, 1024)
    most = max(16, min(4096, int(3.4e10 / (H * K * N))))
    rows = log(1, 64) if rng.random() < 0.4 else log(16, most)
    act, up = rng.choice((("relu", "relu"), ("silu", "none"), ("gelu", "none"), ("relu", "none")))
    return dict(op="gated", rows=rows, H=H, K=K, N=N, act=act, up=up, z=rng.random() < 0.5, half=half, train=train, keep=keep)


# ------------------------------------------------------------------------------ inputs


def _type(case):
    return torch.float16 if case["half"] else torch.bfloat16


def _inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    M = case["rows"]
    if case["op"] == "act8":
        x = rn(M, case["N"]) * torch.exp2(3 * rn(M, 1))  # rows of different sizes
        return dict(x=x.to(dict(bf16=torch.bfloat16, fp16=torch.float16, fp32=torch.float32)[case["type"]]))
    K, N, t = case["K"], case["N"], _type(case)
    if case["op"] == "linear":
        x = rn(M, K)
        if K >= 4 * N:  # the decoder reads products of two rectified projections: sparse, not negative
            x = torch.relu(x) * torch.relu(rn(M, K))
        w = rn(N, K).to(t).t() if case["turned"] else rn(K, N).to(t)
        s = dict(x=x.to(t), w=w * (1.0 / math.sqrt(K)))
        s["b"] = (rn(N) * 0.1).to(t) if case["bias"] else None
        s["r"] = rn(M, N).to(t) if case["residual"] else None
        s["dy"] = rn(M, N).to(t) if case["train"] else None
        wants = ("x", "w", "b")
    else:
        H = case["H"]
        shape = (M, H, N) if H > 1 else (M, N)
        w = lambda: ((rn(H, K, N) if H > 1 else rn(K, N)) * (1.0 / math.sqrt(K))).to(t)  # noqa: E731
        s = dict(x=rn(M, K).to(t), wg=w(), wu=w())
        s["z"] = rn(*((M, H, K) if H > 1 else (M, K))).to(t) if case["z"] else None
        s["dy"] = rn(*shape).to(t) if case["train"] else None
        wants = ("x", "wg", "wu", "z")
    if case["train"]:
        for k in wants:
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    return s


# ------------------------------------------------------------------------------ plain forms


def _held(p, keep, t):
    """The pre-activations that the backward pass goes by: held in the operands' type `t`, or what 8-bit codes stand for."""
    if keep == "16bit":
        return p.to(t).float()
    return _decode(*_encode(p), p.shape[-1]) if keep == "8bit" else p


def _encode(p):
    """e4m3 codes of blocks of 32 values along the last dimension and their scales, powers of two."""
    n = p.shape[-1]
    blocks = torch.nn.functional.pad(p, (0, -n % BLOCK)).unflatten(-1, (-1, BLOCK))
    finite = blocks.isfinite()
    largest = torch.where(finite, blocks.abs(), 0.0).amax(-1, keepdim=True)
    m, e = torch.frexp(largest)
    e = (e - 9 + (m > LARGEST / 512).int()).clamp_min(-126)  # the least one with largest <= 448 2^e
    e = torch.where(largest > 0, e, -126)
    one = torch.ones_like(largest)
    value = torch.where(finite, blocks * torch.ldexp(one, -e), float("nan"))
    return value.to(torch.float8_e4m3fn), torch.ldexp(one, e)


def _decode(codes, scale, n):
    return (codes.float() * scale).flatten(-2)[..., :n]


def _act(p, kind):
    """The activation and its derivative."""
    if kind == "relu":
        on = (p > 0).float()
        return p * on, on
    if kind == "silu":
        s = torch.sigmoid(p)
        return p * s, s * (1 + p * (1 - s))
    if kind == "gelu":
        cdf = 0.5 * (1 + torch.erf(p * math.sqrt(0.5)))
        return p * cdf, cdf + p * torch.exp(-0.5 * p * p) * (1 / math.sqrt(2 * math.pi))
    return p, torch.ones_like(p)


def _linear_plain(s):
    case, t = s["case"], s["x"].dtype
    x, w = s["x"].detach().float(), s["w"].detach().float()
    p = x @ w
    if s["b"] is not None:
        p = p + s["b"].detach().float()
    y = _act(p, case["act"])[0]
    if s["r"] is not None:
        y = y + s["r"].float()
    out = {"y": y.to(t)}
    if case["train"]:
        dp = s["dy"].float() * _act(_held(p, case["keep"], t), case["act"])[1]
        out |= {"dx": (dp @ w.t()).to(t), "dw": (x.t() @ dp).to(t)}
        if s["b"] is not None:
            out["db"] = dp.sum(0).to(t)
    return out


def _gated_plain(s):
    case, t = s["case"], s["x"].dtype
    x, wg, wu = (s[k].detach().float() for k in ("x", "wg", "wu"))
    z = x if s["z"] is None else s["z"].detach().float()
    heads = wg.dim() == 3
    if not heads:
        wg, wu, z = wg[None], wu[None], z[None]
    else:
        z = z.transpose(0, 1) if z.dim() == 3 else z[None]  # [H or 1, M, K]
    g, u = x[None] @ wg, z @ wu
    (f, _), (h, _) = _act(g, case["act"]), _act(u, case["up"])
    join = lambda v: v.transpose(0, 1) if heads else v[0]  # noqa: E731
    out = {"y": join(f * h).to(t).contiguous()}
    if case["train"]:
        (f, df), (h, dh) = _act(_held(g, case["keep"], t), case["act"]), _act(_held(u, case["keep"], t), case["up"])
        dy = s["dy"].float()
        dy = dy.transpose(0, 1) if heads else dy[None]
        dg, du = dy * h * df, dy * f * dh
        dx, dz = (dg @ wg.transpose(1, 2)).sum(0), du @ wu.transpose(1, 2)
        dwg, dwu = x.t()[None] @ dg, z.transpose(1, 2) @ du
        if s["z"] is None:
            dx = dx + dz.sum(0)
        else:
            out["dz"] = join(dz).to(t).contiguous()
        out |= {"dx": dx.to(t), "dwg": (dwg if heads else dwg[0]).to(t), "dwu": (dwu if heads else dwu[0]).to(t)}
    return out


def _act8_plain(s):
    codes, scale = _encode(s["x"].float())
    return {"values": _decode(codes, scale, s["x"].shape[-1]).to(s["x"].dtype)}


# ------------------------------------------------------------------------------ the framework's calls


def _linear_own(s):
    from burn_dragon_b200.ops.feed_forward import linear_act

    case = s["case"]
    y = linear_act(s["x"], s["w"], s["b"], case["act"], residual=s["r"], keep=case["keep"])
    if not case["train"]:
        return {"y": y}
    wants = [k for k in ("x", "w", "b") if s[k] is not None]
    grads = torch.autograd.grad(y, [s[k] for k in wants], s["dy"])
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(wants, grads)}}


def _gated_own(s):
    from burn_dragon_b200.ops.feed_forward import gated_linear

    case = s["case"]
    y = gated_linear(s["x"], s["wg"], s["wu"], z=s["z"], activation=case["act"], up_activation=case["up"], keep=case["keep"])
    if not case["train"]:
        return {"y": y}
    wants = [k for k in ("z", "x", "wg", "wu") if s[k] is not None]
    grads = torch.autograd.grad(y, [s[k] for k in wants], s["dy"])
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(wants, grads)}}


def _act8_own(s):
    from burn_dragon_b200.ops.act8 import pack_activation

    return {"values": pack_activation(s["x"]).unpack()}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _linear_own, "gated": _gated_own, "act8": _act8_own}[op](state)
    return {"linear": _linear_plain, "gated": _gated_plain, "act8": _act8_plain}[op](state)


# ------------------------------------------------------------------------------ what a pass cannot do without


def work(case):
    M, N = case["rows"], case["N"]
    if case["op"] == "act8":  # read, held (33 bytes a block of 32) and read again, written
        size = 4 if case["type"] == "fp32" else 2
        return {"bytes": M * N * 2 * size + 2 * M * (N + -(-N // BLOCK)), "flops": 4 * M * N}
    K = case["K"]
    if case["op"] == "linear":
        x, w, y, b = M * K * 2, K * N * 2, M * N * 2, N * 2 * case["bias"]
        r = y * case["residual"]
        if not case["train"]:
            return {"bytes": x + w + b + r + y, "flops": 2 * M * K * N}
        return {"bytes": 2 * (x + w + b) + r + 2 * y, "flops": 6 * M * K * N}
    H = case["H"]
    x, w, y = M * K * 2, 2 * H * K * N * 2, M * H * N * 2
    x += M * H * K * 2 * case["z"]
    if not case["train"]:
        return {"bytes": x + w + y, "flops": 4 * M * H * K * N}
    return {"bytes": 2 * (x + w + y), "flops": 12 * M * H * K * N}


# ------------------------------------------------------------------------------ the definition, in 64 bits


def _round8(p):
    """Values on the e4m3 grid of their block, nearest, ties to the even code."""
    n = p.shape[-1]
    blocks = torch.cat((p, p.new_zeros(*p.shape[:-1], -n % BLOCK)), -1).reshape(*p.shape[:-1], -1, BLOCK)
    largest = blocks.abs().amax(-1, keepdim=True)
    step = torch.exp2(torch.ceil(torch.log2(largest.clamp_min(2.0 ** -140) / LARGEST)).clamp_min(-126))
    step = torch.where(largest > LARGEST * step, step * 2, torch.where(largest <= LARGEST * step / 2, step / 2, step))
    step = step.clamp_min(2.0 ** -126)
    unit = blocks / step
    grid = torch.exp2(torch.floor(torch.log2(unit.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(unit / grid) * grid * step).reshape(*p.shape[:-1], -1)[..., :n]


_ACTS = {"none": lambda p: p, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}


def _seen(p, case):
    """p with its value replaced by the held one, and its own gradient."""
    if case["keep"] not in ("8bit", "16bit"):
        return p
    at = p.detach()
    return p + ((_round8(at) if case["keep"] == "8bit" else at.to(_type(case)).double()) - at)


def exact(case, seed):
    s = {k: None if v is None else v.detach().double() for k, v in _inputs(case, seed).items()}
    if case["op"] == "act8":
        return {"values": _round8(s["x"])}
    wants = [k for k in ("z", "x", "w", "b", "wg", "wu") if s.get(k) is not None] if case["train"] else []
    for k in wants:
        s[k].requires_grad_(True)
    if case["op"] == "linear":
        p = s["x"] @ s["w"] + (0 if s["b"] is None else s["b"])
        y = _ACTS[case["act"]](p) + (0 if s["r"] is None else s["r"])
        z = _ACTS[case["act"]](_seen(p, case))
    else:
        form = "mk,hkn->mhn" if case["H"] > 1 else "mk,kn->mn"
        other = form if case["H"] == 1 or s["z"] is None else "mhk,hkn->mhn"
        g = torch.einsum(form, s["x"], s["wg"])
        u = torch.einsum(other, s["x"] if s["z"] is None else s["z"], s["wu"])
        f, h = _ACTS[case["act"]], _ACTS[case["up"]]
        y, z = f(g) * h(u), f(_seen(g, case)) * h(_seen(u, case))
    out = {"y": y.detach()}
    if wants:
        out |= {"d" + k: v for k, v in zip(wants, torch.autograd.grad(z, [s[k] for k in wants], s["dy"]))}
    # laid out as run() lays them out
    order = ("y", "dx", "dw", "db") if case["op"] == "linear" else ("y", "dz", "dx", "dwg", "dwu")
    return {k: out[k] for k in order if k in out}
