"""Where adapter_linear must refuse, keep requests apart or give an empty answer."""

import pytest
import torch

from burn_dragon_b200.ops.adapters import AdapterBatch, adapter_linear


def make(M, G=2, H=2, K=16, N=24, r=4, dev="cpu", dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen).to(dev, dtype)  # noqa: E731
    return rn(M, K), rn(H, K, N) * 0.1, rn(G, H, r, K) * K ** -0.5, rn(G, H, r, N) * 0.2


def test_a_plan_of_another_device_is_refused():
    """The plan's indexes decide what is read and written: it has to lie where the operands do."""
    x, w, a, b = make(5)
    elsewhere = AdapterBatch([0, 1], [2, 3], 2, device="meta")
    with pytest.raises(ValueError, match="one device"):
        adapter_linear(x, w, a, b, elsewhere)
    with pytest.raises(ValueError, match="one device"):
        adapter_linear(x, w.to("meta"), a, b, AdapterBatch([0, 1], [2, 3], 2, device="cpu"))


@pytest.mark.gpu
def test_the_binding_refuses_a_plan_of_another_device():
    from burn_dragon_b200 import _ext
    from burn_dragon_b200.ops.gemm import error_word

    x, w, a, b = make(5, dev="cuda", dtype=torch.bfloat16)
    batch = AdapterBatch([0, 1], [2, 3], 2, device="cpu")
    mod, err = _ext.load(), error_word(x.device)
    assert mod.adapter_direct(x, w, a, b, batch.plan, batch.dims, None, 1.0, err) is None
    with pytest.raises(RuntimeError, match="operands' GPU"):
        mod.adapter_forward(x, w, a, b, batch.plan, batch.dims, None, 1.0, err)
