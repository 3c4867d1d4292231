"""Low-rank adapters of many requests at once beside a shared projection (``csrc/adapters.cu``).

``adapter_linear(x, weight, a, b, batch, scale)`` computes, for every row m of a batch that mixes
requests, with g(m) the row's adapter (none: the projection alone)::

    y[m, h] = x[m(, h)] weight[h] + scale[g(m)] (x[m(, h)] a[g(m), h]^T) b[g(m), h]

``weight`` [H, K, N] is frozen and shared (the random scaffold's or any other projection of the
model, laid out as the model keeps it); ``a`` [G, H, r, K] and ``b`` [G, H, r, N] hold G adapters, rows
contiguous. x is [M, K] (every head reads it, as the BDH encoder does) or [M, H, K] (one input per head,
as its y projection). Without heads: weight [K, N], a [G, r, K], b [G, r, N], y [M, N].

A batch is described once by an ``AdapterBatch`` and used for every layer and projection of a
step: prompts, single tokens and any mix of them are rows like any other. The gradients of x, a and b
come from the same kernels; gradients of an adapter that no row uses are zero. An infinity or NaN in one
adapter shows in its own rows and gradients only.

On CUDA x a^T (and dy b^T in the backward pass) is summed in fp32 and rounded to bf16 once, as an operand of the
next product: with the rounding of y itself that makes 0.0018 to 0.0024 of relative error, of which y's is 0.0017.
How a reduction is split depends on the batch, so a request alone answers as among others up to the order of fp32 sums.
"""

from __future__ import annotations

import numpy as np
import torch
from torch.autograd.forward_ad import unpack_dual

from .. import _ext
from .gemm import error_word

TILE = 128  # rows of a product tile
MAX_RANK = 64


class AdapterBatch:
    """The rows of a batch: request i has ``rows[i]`` consecutive rows with adapter ``adapters[i]``
    (-1: none) out of ``n_adapters``. Built on the host, copied to ``device`` once."""

    def __init__(self, adapters, rows, n_adapters: int, device="cuda"):
        ids = np.asarray(adapters, dtype=np.int64).reshape(-1)
        rows = np.asarray(rows, dtype=np.int64).reshape(-1)
        if ids.shape != rows.shape:
            raise ValueError(f"{ids.size} adapters for {rows.size} requests")
        if rows.size and rows.min() < 0:
            raise ValueError("a request cannot have fewer than 0 rows")
        if n_adapters < 1:
            raise ValueError("n_adapters must be at least 1")
        if ids.size and (ids.min() < -1 or ids.max() >= n_adapters):
            raise ValueError(f"adapter ids must be -1 to {n_adapters - 1}")
        of_row = np.repeat(ids, rows)
        self.rows, self.n_adapters = int(of_row.size), int(n_adapters)
        if self.rows >= 1 << 30:
            raise ValueError("too many rows")
        self.device = torch.device(device)
        M, G = self.rows, self.n_adapters
        tiles = -(-M // TILE)
        has = of_row >= 0
        # the distinct adapters of each 128-row tile, and the place ("slot") of a row's among them
        pair = (np.arange(M) // TILE)[has] * G + of_row[has]
        distinct, inverse = np.unique(pair, return_inverse=True)
        tile_ptr = np.searchsorted(distinct, np.arange(tiles + 1) * G)
        row_slot = np.full(M, -1, np.int64)
        row_slot[has] = inverse - tile_ptr[pair // G] if pair.size else inverse
        # rows sorted by adapter, and runs of at most 8 (single tokens) or 32 of them
        order = np.flatnonzero(has)[np.argsort(of_row[has], kind="stable")]
        group = np.searchsorted(of_row[order], np.arange(G + 1))
        count = np.diff(group)
        self._per_chunk = 8 if count.max(initial=0) <= 8 else 32
        runs = -(-count // self._per_chunk)
        g = np.repeat(np.arange(G), runs)
        first = np.arange(runs.sum()) - np.repeat(np.cumsum(runs) - runs, runs)
        start = group[g] + first * self._per_chunk
        chunk = np.stack((start, np.minimum(group[g + 1] - start, self._per_chunk), g), 1)
        by_size = np.argsort(-count, kind="stable")  # the longest first
        flat = np.concatenate([v.reshape(-1) for v in (of_row, row_slot, tile_ptr, distinct % G, order, chunk, group, by_size)])
        self.plan = torch.from_numpy(flat.astype(np.int32)).to(self.device)
        self.dims = [M, G, tiles, int(distinct.size), int(order.size), len(chunk), self._per_chunk]
        self._of_row = of_row

    def adapter_of_row(self) -> torch.Tensor:
        """[M] int64: the adapter of every row, -1 for none."""
        return torch.from_numpy(self._of_row).to(self.device)


def adapter_linear_ref(x, weight, a, b, batch: AdapterBatch, scale=1.0):
    """The same function in elementary operations (the CPU path), differentiable."""
    of = batch.adapter_of_row()
    M, (H, K, N) = x.shape[0], weight.shape
    xh = x[:, None].expand(M, H, K) if x.dim() == 2 else x
    y = torch.einsum("mhk,hkn->mhn", xh, weight)
    out = []
    s = torch.as_tensor(scale, dtype=y.dtype, device=y.device).expand(batch.n_adapters)
    for g in range(batch.n_adapters):
        rows = (of == g).nonzero()[:, 0]
        if rows.numel():
            t = torch.einsum("mhk,hrk->mhr", xh[rows], a[g])
            out.append((rows, s[g] * torch.einsum("mhr,hrn->mhn", t, b[g])))
    for rows, d in out:
        y = y.index_add(0, rows, d.to(y.dtype))
    return y if out else _reach(y, a, b)


def _reach(y, *inputs):
    """``y`` with a gradient of zeros for each of ``inputs``: no row reads them."""
    if not (torch.is_grad_enabled() and any(t.requires_grad for t in inputs)):
        return y
    return y + sum(t[:0].sum() for t in inputs).to(y.dtype)


class _AdapterLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, a, b, batch, scale, scale0):
        y, t = _ext.load().adapter_forward(x, weight, a, b, batch.plan, batch.dims, scale, scale0,
                                           error_word(weight.device))
        ctx.save_for_backward(x, weight, a, b, t, scale)
        ctx.batch, ctx.scale0 = batch, scale0
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, a, b, t, scale = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, da, db = _ext.load().adapter_backward(_rows(dy), x, weight, a, b, t, ctx.batch.plan, ctx.batch.dims, scale,
                                                  ctx.scale0, error_word(weight.device), need[0], need[2], need[3])
        return (dx.view(x.shape) if need[0] else None, None, da if need[2] else None, db if need[3] else None, None, None,
                None)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the kernels read it: 16-byte aligned rows, contiguous in the last dimension."""
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 and s > 0 for s in t.stride()[:-1])
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def adapter_linear(x: torch.Tensor, weight: torch.Tensor, a: torch.Tensor, b: torch.Tensor, batch: AdapterBatch,
                   scale=1.0) -> torch.Tensor:
    """See the module. ``scale``: a number, or an fp32 tensor of one per adapter (on CUDA a constant: one that
    wants a gradient is refused, and so are forward-mode tangents). On CUDA all operands are bf16, K and N multiples of 8, r <= 64; sums are fp32. Tensors
    that are not laid out in aligned rows are copied first."""
    if x.is_cuda:
        tensor = isinstance(scale, torch.Tensor)
        y = _ext.load().adapter_direct(x, weight, a, b, batch.plan, batch.dims, scale if tensor else None,
                                       1.0 if tensor else float(scale), error_word(x.device))
        if y is not None:
            return y
    heads = weight.dim() == 3
    if not heads:
        if weight.dim() != 2 or a.dim() != 3 or b.dim() != 3 or x.dim() != 2:
            raise ValueError("adapter_linear takes weight [H, K, N], a [G, H, r, K], b [G, H, r, N], or all without heads")
        weight, a, b = weight[None], a[:, None], b[:, None]
    if a.dim() != 4 or b.dim() != 4 or x.dim() not in (2, 3):
        raise ValueError("adapter_linear takes x [M, K] or [M, H, K], a [G, H, r, K] and b [G, H, r, N]")
    H, K, N = weight.shape
    G, r = a.shape[0], a.shape[2]
    if a.shape != (G, H, r, K) or b.shape != (G, H, r, N):
        raise ValueError(f"a {tuple(a.shape)} and b {tuple(b.shape)} do not fit a weight of {tuple(weight.shape)}")
    if G != batch.n_adapters:
        raise ValueError(f"the batch was planned for {batch.n_adapters} adapters, not {G}")
    if x.shape[0] != batch.rows or x.shape[-1] != K or (x.dim() == 3 and x.shape[1] != H):
        raise ValueError(f"x {tuple(x.shape)} does not fit {batch.rows} rows and a weight of {tuple(weight.shape)}")
    if weight.requires_grad and torch.is_grad_enabled():
        raise ValueError("the shared projection is frozen: adapter_linear has no gradient for it")
    if isinstance(scale, torch.Tensor) and scale.dim() > 0 and scale.shape != (G,):
        raise ValueError(f"scale must be a number or one value per adapter, got shape {tuple(scale.shape)}")
    if any(t.device != x.device for t in (weight, a, b, batch.plan)):
        raise ValueError("adapter_linear: all operands and the batch must be on one device")
    if not x.is_cuda:
        y = adapter_linear_ref(x, weight, a, b, batch, scale)
        return y if heads else y.view(batch.rows, N)
    if any(t.dtype != torch.bfloat16 for t in (x, weight, a, b)):
        raise TypeError("adapter_linear takes bf16 tensors on CUDA")
    if K % 8 or N % 8 or not 1 <= r <= MAX_RANK:
        raise ValueError(f"adapter_linear takes K and N in multiples of 8 and a rank of 1 to {MAX_RANK}, got K={K} N={N} r={r}")
    tensors = (x, weight, a, b, scale) if isinstance(scale, torch.Tensor) else (x, weight, a, b)
    if any(unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("adapter_linear has no forward-mode derivative on CUDA")
    per, scale0 = None, 1.0
    if isinstance(scale, torch.Tensor):
        if scale.requires_grad and torch.is_grad_enabled():
            raise ValueError("scale is a constant: adapter_linear has no gradient for it on CUDA")
        per = scale if scale.shape == (G,) else scale.expand(G)
        per = per.to(x.device, torch.float32).contiguous()
    else:
        scale0 = float(scale)
    if batch.rows == 0:
        return _reach(x.new_zeros((0, H, N) if heads else (0, N)), x, a, b)
    x, weight, a, b = _rows(x), _rows(weight), _rows(a.contiguous()), _rows(b.contiguous())
    if torch.is_grad_enabled() and (x.requires_grad or a.requires_grad or b.requires_grad):
        y = _AdapterLinear.apply(x, weight, a, b, batch, per, scale0)
    else:
        y = _ext.load().adapter_forward(x, weight, a, b, batch.plan, batch.dims, per, scale0, error_word(x.device))[0]
    return y if heads else y.view(batch.rows, N)
