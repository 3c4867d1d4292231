"""The products of a feed-forward layer with the layer's arithmetic in their epilogue (``csrc/feed_forward.cu``).

``linear_act(x, weight, bias, activation, residual)``::

    y = act(x W + b) + r

``gated_linear(x, w_gate, w_up, ...)``, both projections, their activations and the product in one kernel::

    y = act(x Wg + bg) * up(z Wu + bu)                       z is x unless it is given; up: "none" or "relu"

With heads, as the BDH layer keeps its projections: weights [H, K, N], x and z [M, K] (every head reads it) or [M, H, K],
y [M, H, N]. relu(v E) * relu(a E_v) is ``gated_linear(v, encoder, encoder_v, z=a, up_activation="relu")`` (thresholds are
biases: a number stands for all columns).

``keep`` says what the backward pass goes by: "recompute" keeps the inputs only and computes the pre-activations again,
"16bit" holds them in the operands' type, "8bit" in e4m3 with a scale for 32 columns (``act8``), which its own epilogue
writes. The second is the fastest (a forward and backward pass of 4096 rows: 1024 -> 4096 with GELU 134 us, 155
recomputed, 143 in 8 bits; 256 -> 8192 175, 183, 190) and the default (None too); "recompute" holds the least.

On CUDA the operands are bf16 or fp16 of one type, biases that or fp32; sums are fp32, y and every gradient are rounded once,
and so is dp (the gradient of a pre-activation) as an operand of the next product. Any K and N: sizes that are not
multiples of 8 are padded in a copy. On the CPU the same functions run in plain operations of any floating type.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F
from torch.autograd.forward_ad import unpack_dual

from .. import _ext
from .act8 import decode_ref, encode_ref
from .adapters import _reach, _rows
from .gemm import error_word

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
_UPS = {"none": False, "relu": True}
_KEEPS = {"recompute": 0, "16bit": 1, "8bit": 2}

def activate(p: torch.Tensor, activation: str) -> torch.Tensor:
    if activation == "relu":
        return torch.relu(p)
    if activation == "silu":
        return F.silu(p)
    return F.gelu(p) if activation == "gelu" else p


# ------------------------------------------------------------------------------ CPU


def _held(p: torch.Tensor, keep: str, dtype) -> torch.Tensor:
    """What the backward pass sees of p, with p's own gradient."""
    at = p.detach()
    if keep == "16bit":
        seen = at.to(dtype).to(p.dtype)
    else:
        seen = decode_ref(*encode_ref(at.reshape(-1, p.shape[-1]))).to(p.dtype).view(p.shape)
    return _Forward.apply(seen, p)


class _Forward(torch.autograd.Function):
    """The value of ``y`` with the gradient of ``surrogate``."""

    @staticmethod
    def forward(ctx, y, surrogate):
        return y.detach().clone()

    @staticmethod
    def backward(ctx, dy):
        return None, dy


def _ref(x, z, wg, wu, bg, bu, residual, act, up, keep):
    """The layer [M, H, N] in plain operations, differentiable."""
    low = x.dtype in (torch.bfloat16, torch.float16)
    wide = (lambda t: t.float()) if low else (lambda t: t)
    heads = lambda t: t if t.dim() == 3 else t[:, None].expand(t.shape[0], wg.shape[0], t.shape[1])  # noqa: E731

    def project(t, w, b):
        p = torch.einsum("mhk,hkn->mhn", wide(heads(t)), wide(w))
        return p if b is None else p + (wide(b).to(p.dtype) if isinstance(b, torch.Tensor) else b)

    def finish(g, u):
        y = activate(g, act)
        return y if u is None else y * activate(u, up)

    g = project(x, wg, bg)
    u = None if wu is None else project(x if z is None else z, wu, bu)
    y = finish(g, u)
    if keep in ("16bit", "8bit") and torch.is_grad_enabled() and y.numel() and not (wu is None and act == "none"):
        seen = finish(_held(g, keep, x.dtype), None if u is None else _held(u, keep, x.dtype))
        y = _Forward.apply(y.detach(), seen)
    if residual is not None:
        y = y + wide(residual)
    return y.to(x.dtype)


# ------------------------------------------------------------------------------ CUDA


def _weight(w: torch.Tensor, like: torch.Tensor | None = None) -> torch.Tensor:
    """``w`` [H, K, N] as the kernels read it: K or N contiguous, the other strides multiples of 8 values."""
    def fits(t, inner):
        outer = -3 - inner  # the other one of the last two
        return t.stride(inner) == 1 and t.stride(outer) % 8 == 0 and t.stride(outer) > 0

    ok = (fits(w, -1) or fits(w, -2)) and w.data_ptr() % 16 == 0 and w.stride(0) % 8 == 0 and w.stride(0) > 0
    if not ok:
        w = w.clone(memory_format=torch.contiguous_format)
    if like is not None and (w.stride(-1) == 1) != (like.stride(-1) == 1):  # both projections alike
        w = w.transpose(1, 2).contiguous().transpose(1, 2) if w.stride(-1) == 1 else w.contiguous()
    return w


class _Grow(torch.autograd.Function):
    """[B, R, C] with zeros behind its rows and columns."""

    @staticmethod
    def forward(ctx, t, rows, cols):
        ctx.size = t.shape
        return _ext.load().ff_pad(t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous(), rows, cols)

    @staticmethod
    def backward(ctx, g):
        return g[:, :ctx.size[1], :ctx.size[2]], None, None


def _pad(t, cols: int, rows: int | None = None):
    """``t`` with its last dimension (and the one before) grown by zeros."""
    if not isinstance(t, torch.Tensor):
        return t
    if rows is None:
        if t.shape[-1] == cols:
            return t
        if t.element_size() != 2:
            return F.pad(t, (0, cols - t.shape[-1]))
        return _Grow.apply(t.reshape(1, -1, t.shape[-1]), t.numel() // t.shape[-1] if t.shape[-1] else t.shape[:-1].numel(),
                           cols).view(*t.shape[:-1], cols)
    if t.shape[-2:] == (rows, cols):
        return t
    if t.stride(-1) != 1 and t.stride(-2) == 1:  # as it lies: turned
        return _Grow.apply(t.transpose(-1, -2), cols, rows).transpose(-1, -2)
    return _Grow.apply(t, rows, cols)


def _bias(b, what: str, shape, x):
    if b is None or isinstance(b, (int, float)):
        return
    if not isinstance(b, torch.Tensor) or tuple(b.shape) != shape:
        raise ValueError(f"{what} must be a number or a tensor of {list(shape)}, got {tuple(b.shape) if isinstance(b, torch.Tensor) else b!r}")
    if x.is_cuda and b.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"{what} must be fp32 or of the operands' type, not {b.dtype}")


def _layer(name, x, z, wg, wu, bg, bu, residual, act, up, keep):
    """x, z [M, K] or [M, H, K], weights [H, K, N], biases [H, N], residual [M, H, N]: y [M, H, N]."""
    H, K, N = wg.shape
    M = x.shape[0]
    if act not in ACTIVATIONS:
        raise ValueError(f"{name}: activation {act!r} (one of {', '.join(ACTIVATIONS)})")
    if up not in _UPS:
        raise ValueError(f"{name}: up_activation {up!r} (none or relu)")
    if keep is not None and keep not in _KEEPS:
        raise ValueError(f"{name}: keep {keep!r} (one of {', '.join(_KEEPS)}, or None)")
    keep = keep or "16bit"
    if wu is not None and wu.shape != wg.shape:
        raise ValueError(f"{name}: w_gate {tuple(wg.shape)} and w_up {tuple(wu.shape)} must have one shape")
    for t, what in ((x, "x"), (z, "z")):
        if t is not None and (t.dim() not in (2, 3) or t.shape[0] != M or t.shape[-1] != K or (t.dim() == 3 and t.shape[1] != H)):
            raise ValueError(f"{name}: {what} {tuple(t.shape)} does not fit {M} rows and a weight of {tuple(wg.shape)}")
    if residual is not None and residual.shape != (M, H, N):
        raise ValueError(f"{name}: residual {tuple(residual.shape)} does not fit the output")
    _bias(bg, "bias" if wu is None else "b_gate", (H, N), x)
    _bias(bu, "b_up", (H, N), x)
    tensors = [t for t in (x, z, wg, wu, bg, bu, residual) if isinstance(t, torch.Tensor)]
    if any(t.device != x.device for t in tensors):
        raise ValueError(f"{name}: all operands must be on one device")
    plain = [t for t in (x, z, wg, wu, residual) if t is not None]
    if any(t.dtype != x.dtype for t in plain):
        raise TypeError(f"{name}: all operands must have one type, got {sorted({str(t.dtype) for t in plain})}")
    if not x.is_cuda:
        return _ref(x, z, wg, wu, bg, bu, residual, act, up, keep)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{name} takes bf16 or fp16 tensors on CUDA, not {x.dtype}")
    if any(unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative on CUDA")
    if M == 0 or N == 0 or H == 0:
        return _reach(x.new_zeros((M, H, N)), *tensors)
    K8, N8 = max(8, -(-K // 8) * 8), -(-N // 8) * 8
    if K8 != K or N8 != N:
        x, z, residual = _pad(x, K8), _pad(z, K8), _pad(residual, N8)
        wg, wu, bg, bu = _pad(wg, N8, K8), _pad(wu, N8, K8), _pad(bg, N8), _pad(bu, N8)
    both = [isinstance(b, torch.Tensor) for b in (bg, bu)]
    if all(both) and bg.dtype != bu.dtype:
        bg, bu = bg.float(), bu.float()
    bg0, bu0 = (0.0 if has or b is None else float(b) for has, b in zip(both, (bg, bu)))
    bg, bu = ((_rows(b.contiguous()) if has else None) for has, b in zip(both, (bg, bu)))
    x, wg = _rows(x), _weight(wg)
    z = None if z is None else _rows(z)
    wu = None if wu is None else _weight(wu, wg)
    residual = None if residual is None else _rows(residual)
    if residual is not None:  # heads are for the gated form: one head's rows
        y = _call(x, None, wg[0], None, None if bg is None else bg[0], None, bg0, 0.0, residual[:, 0], act, up, keep)[:, None]
    else:
        y = _call(x, z, wg, wu, bg, bu, bg0, bu0, None, act, up, keep)
    return y if N8 == N else y[..., :N]


def _call(x, z, wg, wu, bg, bu, bg0, bu0, residual, act, up, keep):
    y = _ext.load().ff_call(x, z, wg, wu, bg, bu, bg0, bu0, residual, ACTIVATIONS[act], up == "relu", _KEEPS[keep],
                            error_word(x.device))
    if y is None:
        raise RuntimeError("feed_forward: operands that the kernels cannot read")
    return y


def _direct(x, z, wg, wu, bg, bu, residual, act, up, keep):
    """The call that needs no copy, no padding and no error: its result, or None."""
    if not x.is_cuda or act not in ACTIVATIONS or up not in _UPS or not (keep is None or keep in _KEEPS) or wg.dim() < 2:
        return None
    keep = _KEEPS[keep or "16bit"]
    bg0 = bu0 = 0.0
    if not (bg is None or isinstance(bg, torch.Tensor)):
        bg, bg0 = None, float(bg)
    if not (bu is None or isinstance(bu, torch.Tensor)):
        bu, bu0 = None, float(bu)
    return _ext.load().ff_call(x, z, wg, wu, bg, bu, bg0, bu0, residual, ACTIVATIONS[act], _UPS[up], keep, error_word(x.device))


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias=None, activation: str = "none", *,
               residual: torch.Tensor | None = None, keep: str | None = "16bit") -> torch.Tensor:
    """act(x weight + bias) + residual: x [..., K], weight [K, N] (a ``torch.nn.Linear``'s is ``weight.t()``, which is
    read as it lies), bias a number or [N], residual and result [..., N]. ``activation``: none, relu, silu or gelu."""
    y = _direct(x, None, weight, None, bias, None, residual, activation, "none", keep) if weight.dim() == 2 else None
    if y is not None:
        return y
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[0]:
        raise ValueError(f"linear_act takes x [..., K] and weight [K, N], got {tuple(x.shape)} and {tuple(weight.shape)}")
    K, N = weight.shape
    shape = (*x.shape[:-1], N)
    if residual is not None and tuple(residual.shape) != shape:
        raise ValueError(f"linear_act: residual {tuple(residual.shape)} must have the output's shape {shape}")
    rows = math.prod(x.shape[:-1])
    if isinstance(bias, torch.Tensor):
        if tuple(bias.shape) != (N,):
            raise ValueError(f"linear_act: bias must be a number or [{N}], got {tuple(bias.shape)}")
        bias = bias[None]
    y = _layer("linear_act", x.reshape(rows, K), None, weight[None], None, bias, None,
               None if residual is None else residual.reshape(rows, 1, N), activation, "none", keep)
    return y.reshape(shape)


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate=None, b_up=None, *,
                 z: torch.Tensor | None = None, activation: str = "silu", up_activation: str = "none",
                 keep: str | None = "16bit") -> torch.Tensor:
    """activation(x w_gate + b_gate) * up_activation(z w_up + b_up). Without heads: weights [K, N], x and z [..., K],
    biases [N]; with heads: weights [H, K, N], x and z [M, K] or [M, H, K], biases [H, N], y [M, H, N]."""
    y = _direct(x, z, w_gate, w_up, b_gate, b_up, None, activation, up_activation, keep)
    if y is not None:
        return y
    if w_gate.dim() == 3:
        return _layer("gated_linear", x, z, w_gate, w_up, b_gate, b_up, None, activation, up_activation, keep)
    if w_gate.dim() != 2 or w_up.dim() != 2 or x.dim() < 1 or x.shape[-1] != w_gate.shape[0]:
        raise ValueError(f"gated_linear takes x [..., K] and weights [K, N] or [H, K, N], got {tuple(x.shape)}, "
                         f"{tuple(w_gate.shape)} and {tuple(w_up.shape)}")
    if z is not None and z.shape != x.shape:
        raise ValueError(f"gated_linear: z {tuple(z.shape)} must have x's shape {tuple(x.shape)}")
    K, N = w_gate.shape
    rows = math.prod(x.shape[:-1])
    head = lambda b: b[None] if isinstance(b, torch.Tensor) and b.dim() == 1 else b  # noqa: E731
    y = _layer("gated_linear", x.reshape(rows, K), None if z is None else z.reshape(rows, K), w_gate[None], w_up[None],
               head(b_gate), head(b_up), None, activation, up_activation, keep)
    return y.reshape(*x.shape[:-1], N)
