"""The adapter example on a trained run: texts go through the run's own tokenizer."""

import json
import os

import pytest

from burn_dragon_b200.cli.adapters import main as adapters
from burn_dragon_b200.cli.train import main as train
from burn_dragon_b200.models import adapters as bank
from burn_dragon_b200.utils.tokenizer import BPETokenizer

CFG = os.path.join(os.path.dirname(__file__), "..", "burn_dragon_b200", "configs", "tiny_cpu.toml")
ARGS = ["--text", "the cat the cat", "--text", "abab", "--steps", "1", "--length", "6", "--max-tokens", "3", "--rank", "2"]


def test_a_runs_texts_use_its_tokenizer(tmp_path, monkeypatch, capsys):
    monkeypatch.setenv("BURN_DRAGON_RUN_ROOT", str(tmp_path))
    train(["--config", CFG, "--set", "training.max_iters=1", "--set", "training.checkpoint_interval_iters=1",
           "--set", "model.vocab_size=288", "--run-name", "r"])
    run = json.loads(capsys.readouterr().out.strip().splitlines()[-1])["run_dir"]
    tok = BPETokenizer().train(["the cat the cat the cat"] * 4, 262)
    with open(os.path.join(run, "tokenizer.json"), "w") as f:
        json.dump(tok.to_json(), f)
    seen = []
    step = bank.AdapterBDH.train_step
    monkeypatch.setattr(bank.AdapterBDH, "train_step", lambda self, opt, x, y, *a, **k: seen.append(x) or step(self, opt, x, y, *a, **k))
    adapters(["--run", run, *ARGS])
    line = tok.encode("the cat the cat\n")
    assert max(line) >= 256  # merged tokens, which bytes do not have
    whole = line * 4
    got = seen[0][0].tolist()
    assert any(whole[i:i + 6] == got for i in range(len(line)))
    text = capsys.readouterr().out
    assert "adapter 0: " in text and "adapter 1: " in text
    monkeypatch.setattr(BPETokenizer, "vocab_size", 999)
    with pytest.raises(SystemExit, match="288 tokens, the tokenizer 999"):
        adapters(["--run", run, *ARGS])
