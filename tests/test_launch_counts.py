"""launch_count names the kernels that a call launched, for the bindings where it depends on the arguments."""

import pytest
import torch

from burn_dragon_b200 import _ext
from burn_dragon_b200.ops.adapters import AdapterBatch, adapter_linear
from burn_dragon_b200.ops.sampling import sample_tokens
from burn_dragon_b200.train.optim import AdamWMany


def launched(call):
    before = _ext.launch_count()
    call()
    return _ext.launch_count() - before


@pytest.mark.gpu
def test_calls_count_their_kernels():
    rn = lambda *s: torch.randn(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    x, w, a, b = rn(8, 64), rn(1, 64, 64), rn(2, 1, 4, 64), rn(2, 1, 4, 64)
    _ext.load()
    assert launched(lambda: adapter_linear(x, w, a, b, AdapterBatch([-1], [8], 2))) == 1  # the projection
    assert launched(lambda: adapter_linear(x, w, a, b, AdapterBatch([0], [8], 2))) == 2  # and t
    assert launched(lambda: adapter_linear(x[:0], w, a, b, AdapterBatch([0], [0], 2))) == 0
    long = rn(8, 8192), rn(1, 8192, 64), rn(2, 1, 4, 8192), b
    assert launched(lambda: adapter_linear(*long, AdapterBatch([0], [8], 2))) == 3  # and the sum of its parts
    # t, y; db with u, dx, da: dy has one part of 512 columns
    leaf = x.clone().requires_grad_(True), w, a.clone().requires_grad_(True), b.clone().requires_grad_(True)
    batch = AdapterBatch([0], [8], 2)
    assert launched(lambda: adapter_linear(*leaf, batch).sum().backward()) == 5
    logits, u = torch.randn(3, 50, device="cuda"), torch.rand(3, device="cuda")
    assert launched(lambda: sample_tokens(logits, u)) == 1
    assert launched(lambda: sample_tokens(logits[:0], u[:0])) == 0
    ps = [torch.zeros(3, device="cuda") for _ in range(1500)]
    assert launched(lambda: AdamWMany(ps).step(ps)) == 3  # 640 tensors each
    assert launched(lambda: AdamWMany(ps[:40]).step(ps[:40])) == 1
