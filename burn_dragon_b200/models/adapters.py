"""A bank of low-rank adapters on one frozen BDH model: trained together, served together.

Where a random scaffold (``models.scaffold``) trains one adapter per model, an ``AdapterBank`` keeps G of
them for the three shared projections, W = W_frozen + s A_g^T B_g with s = alpha / r or alpha / sqrt(r), and
a batch may name another adapter for every sequence. ``load_scaffold`` takes adapters over from scaffold models
of one seed, W = gain_g W_seed + s_g A_g^T B_g with the scaling and the gains that they were trained with; the
embedding, the head and the norms are those of the model that ``AdapterBDH`` is given.

``AdapterBDH`` is the BDH forward with the three projections through ``ops.adapters.adapter_linear`` (bf16
operands on CUDA, the plain form on CPU); norms, RoPE and the linear attention are ``models.reference``'s.
``train_step`` updates the adapters of the batch with ``AdamWMany``; ``generate`` serves requests of different
lengths, adapters and sampling settings in one batch (``ops.sampling.sample_tokens``).
"""

from __future__ import annotations

import math

import numpy as np
import torch

from ..ops.adapters import AdapterBatch, adapter_linear
from ..ops.sampling import sample_tokens
from ..train.optim import AdamWMany
from . import reference as R
from .bdh import SCAFFOLD_RECORD
from .generate import feed, hold
from .scaffold import PATHS, scaffold_tensor_cpu
from .state import ModelState

PROJECTIONS = ("encoder", "encoder_v", "decoder")


def bank_shapes(cfg, rank: int) -> dict[str, tuple[int, ...]]:
    """One adapter's matrices; rows contiguous over the projection's inputs (a) and outputs (b)."""
    D, H, Nh = cfg.n_embd, cfg.n_head, cfg.latent_per_head
    return {"encoder.a": (H, rank, D), "encoder.b": (H, rank, Nh), "encoder_v.a": (H, rank, D),
            "encoder_v.b": (H, rank, Nh), "decoder.a": (rank, H * Nh), "decoder.b": (rank, D)}


class AdapterBank:
    """fp32 masters of G adapters and, on CUDA, the bf16 copies that the projections read."""

    def __init__(self, cfg, n_adapters: int, rank: int = 16, alpha: float = 16.0, scaling: str = "rank_stabilized",
                 device="cpu", seed: int = 0):
        if scaling not in ("standard", "rank_stabilized"):
            raise ValueError(f"unknown adapter scaling {scaling!r}")
        self.cfg, self.n_adapters, self.rank = cfg, n_adapters, rank
        self.scale = alpha / rank if scaling == "standard" else alpha / math.sqrt(rank)
        gen = torch.Generator().manual_seed(seed)
        # of adapters from a scaffold, per projection [G]: s / gain (None while all are the bank's own) and the gain of
        # W_seed (None while all are 1)
        self.scales, self.gain = None, None
        self.scaffold = None  # what W_seed was made from, where it is known
        self.master, self.work = {}, {}
        for name, shape in bank_shapes(cfg, rank).items():
            t = torch.zeros(n_adapters, *shape)
            if name.endswith(".a"):  # b starts at zero: a fresh adapter changes nothing
                t.uniform_(-1.0 / math.sqrt(shape[-1]), 1.0 / math.sqrt(shape[-1]), generator=gen)
            self.master[name] = t.to(device)
            cuda = self.master[name].is_cuda
            self.work[name] = self.master[name].bfloat16() if cuda else self.master[name]

    def load_scaffold(self, g: int, source, scale: float | None = None) -> None:
        """Adapter ``g`` from a random-scaffold model, or from the tensors of one by their names in its
        ``state_dict`` (``encoder_a``), in its record (``random_scaffold_adapters.fast.encoder.a``) or
        ``encoder.a``: a [.., in, r], b [.., r, out] and the trained gain. ``scale``: the scaffold's s; by default
        that of the model, of the bank's configuration if that is a scaffold's, or the bank's own.
        ``AdapterBDH`` then takes W_seed, without the model's own adapter, for the frozen projections."""
        cfg = self.cfg
        if isinstance(source, torch.nn.Module):
            if not getattr(source, "scaffold", False):
                raise ValueError("load_scaffold takes a random-scaffold model or its tensors")
            cfg = source.cfg
            parts = {n: source._scaffold_parts(n) for n in PROJECTIONS}
            source = {f"{n}.{k}": t for n in PROJECTIONS for k, t in zip(("a", "b", "gain"), parts[n])}
        rs = cfg.random_scaffold
        if scale is None:
            scale = rs.adapter_scale() if rs.enabled else self.scale
        made = (rs.seed, rs.distribution, cfg.init_std) if rs.enabled else None
        if made and self.scaffold and made != self.scaffold:
            raise ValueError(f"adapters of one bank share W_seed: (seed, distribution, std) {made} is not {self.scaffold}")

        def tensor(name: str):
            proj, part = name.split(".")
            for key in (name, f"{proj}_{part}", f"{SCAFFOLD_RECORD}.{name}"):
                if key in source:
                    return source[key].detach()
            return None

        values, gains = {}, {}
        for name, t in self.master.items():
            v = tensor(name)
            if v is None:
                raise KeyError(f"no {name!r} among the scaffold's tensors")
            v = v.transpose(-1, -2) if name.endswith(".a") else v
            if v.shape != t.shape[1:]:
                raise ValueError(f"{name} is {tuple(v.shape)}, the bank's adapters are {tuple(t.shape[1:])}")
            values[name] = v
        for proj in PROJECTIONS:
            v = tensor(proj + ".gain")
            gains[proj] = 1.0 if v is None else float(v)
            if gains[proj] == 0.0 or not math.isfinite(gains[proj]):
                raise ValueError(f"{proj}: a gain of {gains[proj]} cannot be served beside others")
        like = self.master["encoder.a"]
        if self.scales is None:
            self.scales = {n: like.new_full((self.n_adapters,), self.scale) for n in PROJECTIONS}
        if self.gain is None and any(gain != 1.0 for gain in gains.values()):
            self.gain = {n: like.new_ones(self.n_adapters) for n in PROJECTIONS}
        for name, v in values.items():
            t = self.master[name]
            t[g].copy_(v)
            if self.work[name] is not t:
                self.work[name][g].copy_(t[g])
        for proj, gain in gains.items():
            # y = gain x W_seed + s t b, as the operator computes it: x' W + (s / gain) t' b with x' = gain x
            self.scales[proj][g] = scale / gain
            if self.gain is not None:
                self.gain[proj][g] = gain
        self.scaffold = self.scaffold or made

    def state_dict(self) -> dict:
        """The masters, and how they are applied: ``scale``, and of adapters from a scaffold ``scales``, ``gain`` and
        ``scaffold``."""
        return {**self.master, "scale": self.scale, "scales": self.scales, "gain": self.gain, "scaffold": self.scaffold}

    def load_state_dict(self, sd: dict) -> None:
        """A state of a bank of the same shapes. An ``AdapterBDH`` of this bank takes it over on its next call."""
        for name, t in self.master.items():
            if sd[name].shape != t.shape:
                raise ValueError(f"{name} is {tuple(sd[name].shape)}, the bank's is {tuple(t.shape)}")
        like = self.master["encoder.a"]
        for name, t in self.master.items():
            t.copy_(sd[name])
            if self.work[name] is not t:
                self.work[name].copy_(t)
        own = lambda d: None if d is None else {n: v.to(like.device, torch.float32).clone() for n, v in d.items()}  # noqa: E731
        self.scale, self.scales, self.gain = float(sd["scale"]), own(sd["scales"]), own(sd["gain"])
        self.scaffold = None if sd["scaffold"] is None else tuple(sd["scaffold"])

    def tensors(self, which: dict[str, torch.Tensor]) -> list[torch.Tensor]:
        """Every adapter's own matrices, adapter by adapter."""
        return [which[name][g] for g in range(self.n_adapters) for name in self.master]


class AdapterBDH:
    """BDH with an adapter per sequence; the model's own weights stay as they are."""

    def __init__(self, model, bank: AdapterBank):
        cfg = model.cfg
        if getattr(cfg, "mhc_streams", 1) > 1 or getattr(cfg, "latent_fanout_schedule", None):
            raise ValueError("adapters run on the plain BDH layer: no mHC streams, no latent fan-out")
        if getattr(cfg, "sequence_memory_system", "linear_attention") != "linear_attention":
            raise ValueError("adapters run on the linear-attention memory")
        self.cfg, self.bank = cfg, bank
        with torch.no_grad():
            p = {k: None if v is None else v.detach() for k, v in model.param_dict().items()}
        dev = p["embed"].device
        self.p, self.dtype = p, torch.bfloat16 if dev.type == "cuda" else torch.float32
        self.model = model
        self._freeze()
        self.norm = R.make_norm(cfg.norm_kind, p["norm_gamma"], p["norm_beta"], cfg.norm_eps, p.get("norm_alpha"),
                                p.get("norm_shift"))
        make = {"rope": R.rope_freqs, "pope": R.pope_freqs}.get(cfg.rotary_embedding)
        self.freqs = None if make is None else make(cfg.latent_per_head, cfg.rope_theta, device=dev)
        self.decay = R.decay_vector(cfg.decay_slopes(), device=dev) if cfg.uses_decay() else None

    @torch.no_grad()
    def _freeze(self) -> None:
        """The frozen projections: the model's, or for a scaffold's adapters what they were trained beside."""
        model, bank = self.model, self.bank
        self.on_scaffold = bank.scales is not None
        frozen = {n: self.p[n] for n in PROJECTIONS}
        if self.on_scaffold and getattr(model, "scaffold", False):
            frozen = {n: model.scaffold_base(n) for n in PROJECTIONS}
        if bank.scaffold is not None:
            seed, distribution, std = bank.scaffold
            for n in PROJECTIONS:
                some = min(4096, frozen[n].numel())
                want = scaffold_tensor_cpu(seed, PATHS[n], (some,), std, distribution)
                if not torch.allclose(frozen[n].reshape(-1)[:some].float().cpu(), want, rtol=1e-4, atol=1e-4 * std):
                    raise ValueError(f"{n} is not the W_seed of the scaffold that the adapters were trained on")
        self.weights = {n: frozen[n].to(self.dtype).contiguous() for n in PROJECTIONS}
        self.frozen_for = (self.on_scaffold, bank.scaffold)

    def batch(self, adapters, length: int) -> AdapterBatch:
        """The plan of ``len(adapters)`` sequences of ``length`` tokens."""
        return AdapterBatch(adapters, [length] * len(adapters), self.bank.n_adapters, device=self.p["embed"].device)

    def _linear(self, name: str, x: torch.Tensor, batch: AdapterBatch, work, gains) -> torch.Tensor:
        scale = self.bank.scales[name] if self.on_scaffold else self.bank.scale
        if gains is not None:
            x = x * gains[name].view(-1, *[1] * (x.dim() - 1))
        return adapter_linear(x.to(self.dtype), self.weights[name], work[name + ".a"], work[name + ".b"], batch,
                              scale).float()

    def forward(self, tokens: torch.Tensor, batch: AdapterBatch, state: ModelState | None = None, work=None,
                training: bool = False):
        """Logits [B, T, V] of tokens [B, T], row b T + t of the batch being token t of sequence b.
        ``training``: with the model's dropout."""
        cfg, work, bank = self.cfg, work or self.bank.work, self.bank
        B, T = tokens.shape
        if self.frozen_for != (bank.scales is not None, bank.scaffold):  # adapters of a scaffold came, or went, later
            self._freeze()
        gains = None
        if bank.gain is not None:
            of = batch.adapter_of_row()
            gains = {n: torch.where(of < 0, 1.0, bank.gain[n][of.clamp_min(0)]) for n in PROJECTIONS}
        D, H, Nh = cfg.n_embd, cfg.n_head, cfg.latent_per_head
        pos = state.position if state is not None else 0
        thr, thr_y = cfg.thresholds()
        phases = None
        if self.freqs is not None:
            phases = R.rope_phases(torch.arange(pos, pos + T, device=tokens.device), self.freqs)[None, None]
        v = self.norm(self.p["embed"][tokens])
        rhos = []
        for layer in range(cfg.n_layer):
            x = torch.relu(self._linear("encoder", v.reshape(B * T, D), batch, work, gains) - thr)  # [B T, H, Nh]
            q = x.view(B, T, H, Nh).transpose(1, 2)
            if phases is not None:
                q = R.pope_apply(q, phases) if cfg.rotary_embedding == "pope" else R.rope_apply(q, phases)
            rho0 = state.rhos[layer] if state is not None and state.rhos is not None else None
            a, rho = R.linear_attention_chunked(q, v[:, None], rho0=rho0, decay=self.decay, need_state=state is not None)
            a = self.norm(a).transpose(1, 2).reshape(B * T, H, D)
            y = torch.relu(self._linear("encoder_v", a, batch, work, gains) - thr_y)
            yn = x * y
            if training and cfg.dropout > 0.0:
                yn = torch.nn.functional.dropout(yn, cfg.dropout)
            m = self._linear("decoder", yn.reshape(B * T, H * Nh), batch, work, gains)
            v = self.norm(v + self.norm(m).view(B, T, D))
            rhos.append(rho)
        if state is not None:
            state.rhos = rhos
            state.position += T
        head = self.p["embed"].t() if self.p["lm_head"] is None else self.p["lm_head"]
        return v @ head

    # ---------------------------------------------------------------- training
    def optimizer(self, lr: float = 1e-3, state_bits: int = 32, weight_decay: float = 0.0, seed: int = 0) -> AdamWMany:
        """AdamW over every adapter's matrices; on CUDA it writes the bf16 copies too."""
        bank = self.bank
        cuda = bank.master["encoder.a"].is_cuda
        return AdamWMany(bank.tensors(bank.master), lr=lr, weight_decay=weight_decay, state_bits=state_bits, seed=seed,
                         shadows=bank.tensors(bank.work) if cuda else None)

    def train_step(self, opt: AdamWMany, tokens: torch.Tensor, targets: torch.Tensor, adapters,
                   batch: AdapterBatch | None = None, lr: float | None = None) -> torch.Tensor:
        """One step on sequences [B, T] with the given adapters; those of no sequence are left alone. Dropout
        as in the model's own training: its configuration's rate, unless the model is in evaluation mode.
        ``batch``: the plan of an earlier step with the same adapters. Returns the mean loss."""
        bank = self.bank
        batch = batch or self.batch(adapters, tokens.shape[1])
        if not np.array_equal(batch._of_row, np.repeat(np.asarray(adapters, dtype=np.int64), tokens.shape[1])):
            raise ValueError("the batch was planned for other adapters or another length")
        names = list(bank.master)
        work = {n: t.detach().requires_grad_(True) for n, t in bank.work.items()}
        loss = R.cross_entropy(self.forward(tokens, batch, work=work, training=self.model.training), targets)
        grads = dict(zip(names, torch.autograd.grad(loss, [work[n] for n in names])))
        used = {int(g) for g in adapters}
        opt.step([grads[n][g] if g in used else None for g in range(bank.n_adapters) for n in names], lr=lr)
        return loss.detach()

    # ---------------------------------------------------------------- serving
    @torch.no_grad()
    def generate(self, prompts: list[list[int]], adapters, max_new_tokens: int, temperature=1.0, top_k=0, top_p=1.0,
                 min_p=0.0, seed: int = 0) -> tuple[list[list[int]], list[list[float]]]:
        """Continuations of prompts of different lengths, each with its adapter (-1: none) and settings (numbers,
        or one value per request), and the tokens' log-probabilities. Every row advances at the same
        position; one still inside its prompt takes its next prompt token. A request whose logits leave
        nothing to draw from answers -1 (log-probability -inf) from there on; the others go on."""
        if len(prompts) != len(adapters) or not prompts or any(not p for p in prompts):
            raise ValueError("one adapter per prompt, and no empty prompts")
        if max_new_tokens <= 0:
            return [[] for _ in prompts], [[] for _ in prompts]
        dev = self.p["embed"].device
        lens = torch.tensor([len(p) for p in prompts], device=dev)
        width, shared = int(lens.max()), int(lens.min())
        table = torch.tensor([p + [0] * (width - len(p)) for p in prompts], device=dev)
        setting = lambda v, dt: torch.as_tensor(v, dtype=dt, device=dev).expand(len(prompts)).contiguous()  # noqa: E731
        settings = [setting(temperature, torch.float32), setting(top_k, torch.int32), setting(top_p, torch.float32),
                    setting(min_p, torch.float32)]
        gen = torch.Generator(device=dev).manual_seed(seed)
        state = ModelState.empty()
        logits = self.forward(table[:, :shared], self.batch(adapters, shared), state)[:, -1]
        step = self.batch(adapters, 1)  # one plan for all single-token steps
        tokens, logprobs = [], []
        nxt = None
        for pos in range(shared, width + max_new_tokens):
            drawn, lp = sample_tokens(logits.contiguous(), torch.rand(len(prompts), generator=gen, device=dev), *settings)
            nxt = torch.where(lens > pos, table[:, min(pos, width - 1)], hold(drawn, nxt))
            tokens.append(nxt)
            logprobs.append(torch.where(nxt < 0, float("-inf"), lp))
            if pos + 1 < width + max_new_tokens:
                logits = self.forward(feed(nxt)[:, None], step, state)[:, -1]
        host_t = torch.stack(tokens, 1).tolist()
        host_l = torch.stack(logprobs, 1).tolist()
        start = [len(p) - shared for p in prompts]
        return ([t[s:s + max_new_tokens] for t, s in zip(host_t, start)],
                [t[s:s + max_new_tokens] for t, s in zip(host_l, start)])
