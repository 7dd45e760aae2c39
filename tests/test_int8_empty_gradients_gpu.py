"""Gradients of the integer linear layer where a dimension is empty, by both halves of the binding."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("half", ["native", "python"])
@pytest.mark.parametrize("lead,n,k", [((0,), 5, 16), ((4,), 0, 16), ((4,), 6, 0), ((2, 3), 6, 0), ((2, 3), 0, 8), ((0, 3), 4, 8), ((0,), 0, 0)])
def test_gradients(cuda_device, monkeypatch, half, lead, n, k):
    from actnn_b200 import _lib, ops
    if half == "python":
        monkeypatch.setattr(_lib, "_native", False)
    x, w, b = (torch.randn(*s, device="cuda", requires_grad=True) for s in (lead + (k,), (n, k), (n,)))
    y = ops.int8_linear.apply(x, w, b)
    assert y.shape == lead + (n,)
    dy = torch.randn_like(y)
    y.backward(dy)
    assert x.grad.shape == x.shape and w.grad.shape == w.shape
    assert not x.grad.any() or n > 0 and k > 0
    assert not w.grad.any()
    want = dy.double().reshape(torch.Size(lead).numel(), n).sum(0)
    assert torch.allclose(b.grad.double(), want, rtol=0, atol=1e-6 * (1 + float(dy.abs().sum())))
