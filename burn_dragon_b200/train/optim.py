"""Fused AdamW over the flat parameter store, plus learning-rate schedules.

AdamW with decoupled weight decay, beta (0.9, 0.999) defaults and optional global
grad-norm clipping or, when no norm is set, element-wise value clipping (burn_dragon_train/src/config/optimizer.rs:6-460). On CUDA one kernel
updates the fp32 master weights, both moments and the bf16 GEMM shadow in a single
pass over the flat buffers; the clipping coefficient stays on the device.
LR schedules mirror burn_dragon_train/src/train/pipeline/schedule.rs:6-392.
"""

from __future__ import annotations

import math

import torch

from .. import _ext


def lr_at(step: int, base_lr: float, schedule: dict | None, max_iters: int) -> float:
    """Constant / cosine(warmup, min) / linear / exponential / step / noam."""
    sched = dict(schedule or {"type": "constant"})
    kind = sched.get("type", "constant")
    warm = int(sched.get("warmup_iters", 0))
    if warm and step < warm:
        return base_lr * (step + 1) / warm
    if kind == "constant":
        return base_lr
    t = max(0, step - warm)
    span = max(1, max_iters - warm)
    min_lr = float(sched.get("min_lr", 0.0))
    if kind == "cosine":
        c = 0.5 * (1.0 + math.cos(math.pi * min(1.0, t / span)))
        return min_lr + (base_lr - min_lr) * c
    if kind == "linear":
        return base_lr + (min_lr - base_lr) * min(1.0, t / span)
    if kind == "exponential":
        return base_lr * float(sched.get("gamma", 0.999)) ** t
    if kind == "step":
        return base_lr * float(sched.get("gamma", 0.1)) ** (t // int(sched.get("step_size", 1000)))
    if kind == "noam":
        d = float(sched.get("model_dim", 256))
        s = step + 1
        return base_lr * d ** -0.5 * min(s ** -0.5, s * max(1, warm) ** -1.5)
    raise ValueError(f"unknown lr schedule {kind!r}")


class FusedAdamW:
    """AdamW over ``ParamStore`` flat buffers (a boolean mask selects trainable elements)."""

    def __init__(self, store, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1,
                 grad_clip_norm: float | None = None, grad_clip_value: float | None = None):
        self.store = store
        self.clip_value = grad_clip_value if grad_clip_norm is None else None
        self.lr = lr
        self.b1, self.b2 = betas
        self.eps = eps
        self.wd = weight_decay
        self.clip = grad_clip_norm
        self.m = torch.zeros_like(store.data)
        self.v = torch.zeros_like(store.data)
        self.t = 0
        self._scratch = torch.zeros(4, dtype=torch.float32, device=store.data.device)
        # {lr, 1-b1^t, 1-b2^t} on the device, so a captured step reads this step's values
        self._hyper = torch.zeros(4, dtype=torch.float32, device=store.data.device)
        # pageable on purpose: the copy from pageable memory is staged before copy_ returns,
        # so the next step may overwrite this buffer while the GPU still lags behind
        self._hyper_host = torch.zeros(4, dtype=torch.float32)

    def state_dict(self) -> dict:
        return {"m": self.m, "v": self.v, "t": self.t, "lr": self.lr}

    def load_state_dict(self, sd: dict) -> None:
        self.m.copy_(sd["m"])
        self.v.copy_(sd["v"])
        self.t = int(sd["t"])

    def grad_norm(self) -> torch.Tensor:
        return self._scratch[1]

    def prepare(self, lr: float | None = None) -> None:
        """Advance the step counter and stage this step's scalars on the device."""
        self.t += 1
        self._lr_now = self.lr if lr is None else lr
        self._hyper_host[0] = self._lr_now
        self._hyper_host[1] = 1.0 - self.b1 ** self.t
        self._hyper_host[2] = 1.0 - self.b2 ** self.t
        if self.store.data.is_cuda:
            self._hyper.copy_(self._hyper_host, non_blocking=True)

    @torch.no_grad()
    def apply(self) -> None:
        """The update itself (device work only on CUDA; safe to capture in a CUDA graph)."""
        s = self.store
        if self.clip_value is not None:  # burn's GradientClipping::Value: clamp every element
            s.grad.clamp_(-self.clip_value, self.clip_value)
        if s.data.is_cuda:
            mod = _ext.load()
            gscale = None
            if self.clip is not None:
                mod.grad_clip_coef(s.grad, self._scratch, float(self.clip))
                gscale = self._scratch[2:3]
            mod.adamw(s.data, s.grad, self.m, self.v, s.shadow, 0.0, self.b1, self.b2, self.eps, self.wd, 1.0, 1.0,
                      gscale, self._hyper)
            return
        lr = self._lr_now
        bc1, bc2 = float(self._hyper_host[1]), float(self._hyper_host[2])
        g = s.grad
        if self.clip is not None:
            norm = g.norm()
            self._scratch[1] = norm
            g = g * torch.clamp(self.clip / (norm + 1e-6), max=1.0)
        self.m.mul_(self.b1).add_(g, alpha=1 - self.b1)
        self.v.mul_(self.b2).addcmul_(g, g, value=1 - self.b2)
        s.data.mul_(1 - lr * self.wd)
        s.data.addcdiv_(self.m / bc1, (self.v / bc2).sqrt_().add_(self.eps), value=-lr)

    @torch.no_grad()
    def step(self, lr: float | None = None) -> None:
        self.prepare(lr)
        self.apply()


BLOCK = 256  # values of a state that share one 8-bit scale


def _e4m3_stochastic(x: torch.Tensor, bits16: torch.Tensor, floor: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """[n * 256] values -> (e4m3 codes, one scale per 256), as csrc/adamw_many.cu rounds them."""
    b = x.view(-1, BLOCK)
    amax = b.abs().amax(1, keepdim=True)
    fine = (amax >= 2.0 ** -110) & (amax < math.inf)
    scale = torch.where(fine, amax * 2.0 ** -8, torch.where(amax < 2.0 ** -110, torch.zeros_like(amax), amax))
    inverse = torch.where(fine, 256.0 / amax, torch.zeros_like(amax))
    # multiplied by 2^-120 the e4m3 grid is bits 20 and up of the fp32 pattern, denormals included
    y = (b.abs() * inverse) * 2.0 ** -120
    code = (y.view(torch.int32) + (bits16.view(-1, BLOCK) << 4).to(torch.int32)) >> 20
    if floor:
        code = torch.where(b > 0, code.clamp_min(1), code)
    code = torch.where(b < 0, code + 128, code) * fine
    return code.to(torch.uint8).view(torch.float8_e4m3fn).reshape(-1), scale[:, 0]


class AdamWMany:
    """AdamW over many tensors in one launch, e.g. the adapters of an ``AdapterBank``.

    ``params``: contiguous fp32 or bf16 tensors of one device; ``shadows``: none, or a bf16
    working copy of each that the step writes too. ``state_bits`` 32 keeps both moments in fp32, 8
    keeps them as e4m3 codes with one fp32 scale per 256 values (a quarter of the state and
    of its traffic), rounded stochastically from ``seed``, the step and the index, so that a
    step of v by a thousandth of itself is kept on average and a run repeats bit for bit.

    ``state``: ``m`` and ``v`` (and ``m_scale`` / ``v_scale``), every tensor padded to blocks of 256
    values in the order of ``params``. A tensor whose gradient is None is left alone, and its moments are
    corrected for the steps that it has had itself (``steps``), not for those of the others (``t``): an adapter
    that joins late or is trained rarely moves as it would alone. The step counts and the learning rate are
    arguments of the launch, so a captured CUDA graph would repeat one step; ``FusedAdamW`` keeps
    them on the device for that."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.1,
                 state_bits: int = 32, shadows=None, seed: int = 0):
        self.params = [p.detach() for p in params]
        if not self.params:
            raise ValueError("AdamWMany needs at least one tensor")
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        dev = self.params[0].device
        self.shadows = [] if shadows is None else list(shadows)
        if self.shadows and len(self.shadows) != len(self.params):
            raise ValueError("no shadows, or one per tensor")
        for p in self.params:
            if p.device != dev or not p.is_contiguous() or p.dtype not in (torch.float32, torch.bfloat16):
                raise ValueError("AdamWMany takes contiguous fp32 or bf16 tensors on one device")
        for p, s in zip(self.params, self.shadows):
            if s.device != dev or not s.is_contiguous() or s.dtype != torch.bfloat16 or s.numel() != p.numel():
                raise ValueError("a shadow is a contiguous bf16 tensor of its tensor's size")
        self.lr, (self.b1, self.b2), self.eps, self.wd = lr, betas, eps, weight_decay
        self.state_bits, self.seed, self.t = state_bits, int(seed), 0
        self._steps = torch.zeros(len(self.params), dtype=torch.int64)  # on the host; the launch reads and advances it
        sizes = [-(-p.numel() // BLOCK) for p in self.params]
        self.block0 = [0]
        for n in sizes:
            self.block0.append(self.block0[-1] + n)
        total = self.block0[-1]
        self.owner = torch.repeat_interleave(torch.arange(len(sizes), dtype=torch.int32),
                                             torch.tensor(sizes)).to(dev)
        kind = torch.float8_e4m3fn if state_bits == 8 else torch.float32
        self.state = {k: torch.zeros(total * BLOCK, dtype=kind, device=dev) for k in ("m", "v")}
        if state_bits == 8:
            self.state |= {k: torch.zeros(total, device=dev) for k in ("m_scale", "v_scale")}

    @property
    def steps(self) -> list[int]:
        """The steps that each tensor has had."""
        return self._steps.tolist()

    def state_dict(self) -> dict:
        return {**self.state, "t": self.t, "steps": self.steps, "lr": self.lr, "seed": self.seed}

    def load_state_dict(self, sd: dict) -> None:
        """A state without ``steps``: every tensor has had all ``t`` steps."""
        for k, t in self.state.items():
            if sd[k].dtype != t.dtype or sd[k].shape != t.shape:
                raise ValueError(f"state {k!r} is {tuple(sd[k].shape)} {sd[k].dtype}, not {tuple(t.shape)} {t.dtype}")
        steps = [int(n) for n in sd.get("steps", [sd["t"]] * len(self.params))]
        if len(steps) != len(self.params):
            raise ValueError(f"{len(steps)} step counts for {len(self.params)} tensors")
        for k, t in self.state.items():
            t.copy_(sd[k])
        self.t = int(sd["t"])
        self._steps.copy_(torch.tensor(steps))
        self.seed = int(sd.get("seed", self.seed))

    def moments(self, i: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The first and second moment of tensor ``i`` in fp32, in its shape."""
        lo, hi = self.block0[i], self.block0[i + 1]
        p, out = self.params[i], []
        for k in ("m", "v"):
            x = self.state[k][lo * BLOCK:hi * BLOCK].float().view(-1, BLOCK)
            if self.state_bits == 8:
                x = x * self.state[k + "_scale"][lo:hi, None]
            out.append(x.reshape(-1)[:p.numel()].view(p.shape))
        return out[0], out[1]

    @torch.no_grad()
    def step(self, grads, lr: float | None = None, grad_scale: torch.Tensor | None = None) -> None:
        """One step. ``grads``: a gradient (fp32 or bf16) or None per tensor; ``grad_scale``: an
        fp32 device scalar that multiplies them all (a clipping coefficient)."""
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"{len(grads)} gradients for {len(self.params)} tensors")
        t = self.t + 1
        lr = self.lr if lr is None else lr
        key = (self.seed * 0x9E3779B1 + t * 0x85EBCA77) & 0xFFFFFFFF
        if self.state["m"].is_cuda:
            grads = [g if g is None or g.is_contiguous() else g.contiguous() for g in grads]
            _ext.load().adamw_many(self.params, grads, self.shadows, self.block0, self.owner, self.state["m"],
                                   self.state["v"], self.state.get("m_scale"), self.state.get("v_scale"), lr, self.b1,
                                   self.b2, self.eps, self.wd, self._steps, key, grad_scale)
        else:
            for p, g in zip(self.params, grads):
                if g is not None and g.numel() != p.numel():
                    raise ValueError("a gradient has its tensor's size")
            for i, (p, g) in enumerate(zip(self.params, grads)):
                if g is not None:
                    n = int(self._steps[i]) + 1
                    self._step_cpu(i, p, g, lr, 1.0 - self.b1 ** n, 1.0 - self.b2 ** n, key, grad_scale)
                    self._steps[i] = n
        self.t = t

    def _step_cpu(self, i, p, g, lr, bc1, bc2, key, grad_scale) -> None:
        blocks = slice(self.block0[i], self.block0[i + 1])
        values = slice(blocks.start * BLOCK, blocks.stop * BLOCK)
        n = p.numel()
        g = torch.nn.functional.pad(g.reshape(-1).float(), (0, -n % BLOCK))
        g = g if grad_scale is None else g * grad_scale
        m, v = (self.state[k][values].float() for k in ("m", "v"))
        if self.state_bits == 8:
            m, v = ((x.view(-1, BLOCK) * self.state[k][blocks, None]).view(-1)
                    for x, k in ((m, "m_scale"), (v, "v_scale")))
        m = m * self.b1 + g * (1 - self.b1)
        v = v * self.b2 + (g * g) * (1 - self.b2)
        q = p.reshape(-1).float() * (1 - lr * self.wd) - lr * ((m / bc1) / ((v / bc2).sqrt() + self.eps))[:n]
        p.view(-1).copy_(q)
        if self.shadows:
            self.shadows[i].view(-1).copy_(q)
        if self.state_bits == 8:
            h = (torch.arange(values.start, values.stop) * 0x9E3779B1 + key) & 0xFFFFFFFF
            h = ((h ^ (h >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
            h = ((h ^ (h >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
            h = h ^ (h >> 16)
            m, self.state["m_scale"][blocks] = _e4m3_stochastic(m, h & 0xFFFF, False)
            v, self.state["v_scale"][blocks] = _e4m3_stochastic(v, h >> 16, True)
        self.state["m"][values], self.state["v"][values] = m, v
