"""Activations held in 8 bits between the forward and the backward pass (``csrc/act8.cu``).

Values in runs of 32 along the last dimension (the last run of a row may be shorter) share a scale 2^e and are e4m3
codes of x 2^-e, with e the least integer >= -126 for which the largest finite |x| of the run is at most 448 2^e:
nothing saturates, and a value comes back within 2^-4 of itself, or within 2^-10 2^e where it is below 2^-6 2^e
(about 2^-15 of the largest). A value that is not finite comes back as NaN. 33 bytes hold 32 values.

``pack_activation(x)`` packs one tensor; ``activations_in_8bit()`` is a context in which autograd keeps what it saves for
the backward pass in this form, whatever operation saves it. ``feed_forward`` packs its pre-activations in the
product's own epilogue instead (``keep="8bit"``).
"""

from __future__ import annotations

from contextlib import contextmanager

import torch

from .. import _ext

BLOCK = 32
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def encode_ref(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes [R, N] and exponents + 127 [R, ceil(N / 32)] of rows [R, N], uint8, in elementary operations (the CPU path)."""
    R, N = x.shape
    if x.numel() == 0:
        return x.new_empty((R, N), dtype=torch.uint8), x.new_empty((R, -(-N // BLOCK)), dtype=torch.uint8)
    v = torch.nn.functional.pad(x.float(), (0, -N % BLOCK)).view(R, -1, BLOCK)
    finite = v.isfinite()
    largest = torch.where(finite, v.abs(), 0.0).amax(-1, keepdim=True)
    m, e = torch.frexp(largest)
    e = torch.where(largest > 0, (e - 9 + (m > 0.875).int()).clamp_min(-126), -126)
    codes = torch.where(finite, torch.ldexp(v, -e), float("nan")).to(torch.float8_e4m3fn).view(torch.uint8)
    codes = torch.where(finite, codes, torch.tensor(0x7F, dtype=torch.uint8, device=x.device))
    return codes.view(R, -1)[:, :N].contiguous(), (e + 127).to(torch.uint8)[..., 0]


def decode_ref(codes: torch.Tensor, exponents: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """The values that ``encode_ref``'s codes stand for; rounding up never carries one past the type's largest number."""
    R, N = codes.shape
    if codes.numel() == 0:
        return codes.new_empty((R, N), dtype=dtype)
    v = codes.view(torch.float8_e4m3fn).float()
    e = exponents.int() - 127
    scale = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)
    v = v * scale.repeat_interleave(BLOCK, 1)[:, :N]
    top = min(torch.finfo(dtype).max, torch.finfo(torch.float32).max)
    return torch.where(v.isnan(), v, v.clamp(-top, top)).to(dtype)


class PackedActivation:
    """A tensor's values in 8 bits: ``codes`` [rows, N], ``exponents`` [rows, ceil(N / 32)], and what it was."""

    __slots__ = ("codes", "exponents", "shape", "dtype")

    def __init__(self, codes, exponents, shape, dtype):
        self.codes, self.exponents, self.shape, self.dtype = codes, exponents, tuple(shape), dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()

    def unpack(self) -> torch.Tensor:
        """The values, in the packed tensor's shape and type."""
        if self.codes.is_cuda:
            return _ext.load().act8_unpack(self.codes, self.exponents, self.shape, _TYPES[self.dtype])
        return decode_ref(self.codes, self.exponents, self.dtype).view(self.shape)


def pack_activation(x: torch.Tensor) -> PackedActivation:
    """Packs an fp32, bf16 or fp16 tensor (a copy of one that is not contiguous). No graph is kept."""
    if x.dtype not in _TYPES:
        raise TypeError(f"pack_activation takes fp32, bf16 or fp16 values, not {x.dtype}")
    if x.is_cuda:
        codes, exponents = _ext.load().act8_pack(x)
    else:
        rows = x.detach()
        codes, exponents = encode_ref(rows.reshape(-1, rows.shape[-1] if x.dim() else 1) if x.numel() else rows.reshape(0, 1))
    return PackedActivation(codes, exponents, x.shape, x.dtype)


@contextmanager
def activations_in_8bit(min_values: int = 4096, exclude=()):
    """Within it, autograd holds what operations save for the backward pass in 8 bits: fp32, bf16 and fp16 tensors of
    at least ``min_values`` values in rows of 32 or more. Leaves (parameters, inputs) and views of them stay as they
    are, and so do ``exclude``'s tensors: weights that are cast on the way belong there. The backward pass may run
    outside. A gradient then goes by values within 2^-4 of what they were, and a positive value below 2^-10 of
    its run's scale reads as 0 (relu's mask)."""
    kept = [t.untyped_storage() for t in exclude]  # held here, so that no other storage can take an address of theirs
    kept = {st.data_ptr(): st for st in kept}

    def pack(t: torch.Tensor):
        source = t if t._base is None else t._base
        if (t.dtype not in _TYPES or t.layout != torch.strided or t.dim() == 0 or t.shape[-1] < BLOCK
                or t.numel() < min_values or source.is_leaf and source.requires_grad
                or isinstance(source, torch.nn.Parameter) or t.untyped_storage().data_ptr() in kept):
            return t
        return pack_activation(t)

    def unpack(v):
        return v.unpack() if isinstance(v, PackedActivation) else v

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        yield
