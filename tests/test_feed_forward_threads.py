"""The feed-forward operators from threads that have launched nothing on the GPU yet."""

import threading

import pytest
import torch

from burn_dragon_b200.ops.feed_forward import linear_act


@pytest.mark.gpu
def test_a_backward_pass_as_the_first_launch_of_a_thread():
    """Only cached memory and tensor maps before the first launch: the driver's encoder wants a context of the thread's own."""
    x = torch.randn(4, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(64, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    want = torch.autograd.grad(linear_act(x, w, 0.5, "gelu", keep="recompute").float().sum(), (x, w))
    got, failed = [], []

    def work():
        try:
            got.append(linear_act(x.detach(), w.detach(), 0.5, "gelu"))
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    with torch.no_grad():
        y = linear_act(x, w, 0.5, "gelu")
    del_ = torch.empty(4, 256, device="cuda", dtype=torch.bfloat16)
    del del_  # the thread's output comes from the cache
    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert not failed and torch.equal(got[0], y)
    again = torch.autograd.grad(linear_act(x, w, 0.5, "gelu", keep="recompute").float().sum(), (x, w))
    assert all(torch.equal(a, b) for a, b in zip(want, again))
