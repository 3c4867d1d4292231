"""Adapters of many requests, from training to answers, on one frozen BDH model.

Each given text gets an adapter of its own; one batch per step trains them together
(``AdapterBDH.train_step``), then one batch of prompts, each with its adapter, is continued.

  python -m burn_dragon_b200.cli.adapters --text "the quick brown fox" --text "0123456789" [--run runs/language/cuda/NAME]
         [--steps 200] [--rank 16] [--state-bits 8] [--max-tokens 32] [--temperature 0.8 --top-k 40 --top-p 0.95 --min-p 0.05]

Without ``--run`` the frozen model is the tiny byte configuration with random weights. A run's texts go through
its own ``tokenizer.json`` (bytes where it has none).
"""

from __future__ import annotations

import argparse
import os

import torch

from ..config import DragonConfig, training_config_from_dict
from ..models.adapters import AdapterBank, AdapterBDH
from ..models.bdh import BDH
from ..utils.tokenizer import ByteTokenizer, load_tokenizer


def main(argv=None) -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--text", action="append", required=True, help="one training text (and adapter) each")
    ap.add_argument("--run", default=None, help="run directory of the frozen model")
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--length", type=int, default=64, help="tokens of a training sequence")
    ap.add_argument("--lr", type=float, default=3e-3)
    ap.add_argument("--rank", type=int, default=16)
    ap.add_argument("--state-bits", type=int, choices=(8, 32), default=32)
    ap.add_argument("--max-tokens", type=int, default=32)
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--min-p", type=float, default=0.0)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)
    dev = torch.device("cuda", 0) if torch.cuda.is_available() else torch.device("cpu")
    tok = ByteTokenizer()
    if a.run:
        from ..train.checkpoint import RunDir

        run = RunDir(a.run)
        model = BDH(training_config_from_dict(run.read_json("training_config.json")).model, device=dev)
        run.load(None, model)
        path = os.path.join(a.run, "tokenizer.json")
        tok = load_tokenizer(path) if os.path.exists(path) else tok
    else:
        cfg = DragonConfig.tiny()
        cfg.init_std = 0.1  # a random head that can tell bytes apart
        model = BDH(cfg, device=dev, seed=a.seed)
    if model.cfg.vocab_size < tok.vocab_size:
        raise SystemExit(f"the model has {model.cfg.vocab_size} tokens, the tokenizer {tok.vocab_size}")
    G = len(a.text)
    net = AdapterBDH(model, AdapterBank(model.cfg, G, rank=a.rank, device=dev, seed=a.seed))
    opt = net.optimizer(lr=a.lr, state_bits=a.state_bits, seed=a.seed)
    lines = [tok.encode(t + "\n") for t in a.text]
    data = [torch.tensor(ids * (2 + (a.length + 1) // len(ids)), dtype=torch.long) for ids in lines]
    gen = torch.Generator().manual_seed(a.seed)
    plan = net.batch(range(G), a.length)
    for step in range(a.steps):
        rows = []
        for d in data:
            at = int(torch.randint(0, len(d) - a.length, (1,), generator=gen))
            rows.append(d[at:at + a.length + 1])
        xy = torch.stack(rows).to(dev)
        loss = net.train_step(opt, xy[:, :-1], xy[:, 1:], range(G), batch=plan)
        if step % 50 == 0 or step + 1 == a.steps:
            print(f"step {step}: loss {float(loss):.4f}")
    prompts = [ids[:max(1, len(ids) // 2)] for ids in map(tok.encode, a.text)]
    out, logprobs = net.generate(prompts, list(range(G)), a.max_tokens, a.temperature, a.top_k, a.top_p, a.min_p, a.seed)
    for g, (p, o, lp) in enumerate(zip(prompts, out, logprobs)):
        if -1 in o:
            print(f"adapter {g}: no token to draw after {o.index(-1)} tokens: the logits are NaN or -inf")
            continue
        text = tok.decode([t for t in p + o if t < tok.vocab_size])  # a model may have more tokens than its tokenizer
        print(f"adapter {g}: {text!r} (mean log-probability {sum(lp) / max(len(lp), 1):.3f})")


if __name__ == "__main__":
    main()
