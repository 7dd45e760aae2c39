"""The identity needs nothing of its input for the backward pass, and keeps nothing."""
import pytest
import torch

from test_swap_token_inputs_gpu import held

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("half", ["native", "python"])
@pytest.mark.parametrize("level", ["L3", "L0", "L4", "swap"])
def test_bytes_and_gradient(cuda_device, monkeypatch, level, half):
    import actnn_b200 as actnn
    from actnn_b200 import _lib, ops
    if half == "python":
        monkeypatch.setattr(_lib, "_native", False)
    actnn.set_optimization_level(level)
    leaf = torch.randn(512, 1000, device="cuda", requires_grad=True)
    before = held()
    h = leaf * 1
    y = ops.activation.apply(h, "none")
    assert torch.equal(y, h)
    del h
    assert held() - before == y.numel() * 4
    dy = torch.randn_like(y)
    y.backward(dy)
    assert torch.equal(leaf.grad, dy)
    x = torch.randn(6, 10, device="cuda", requires_grad=True)          # the gated form keeps both halves: each one's gradient is the other
    y = ops.glu.apply(x, "none")
    y.sum().backward()
    assert x.grad.shape == x.shape and bool((x.grad != 0).any())
