"""The backward pass of the norms around a residual branch as a function of its own: calls that make no sense (no GPU needed)."""
import pytest
import torch


def test_no_gradient_at_all():
    from actnn_b200.cpp_extension import residual_norm
    x, st = torch.zeros(4, 16), torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="one of grad_r and grad_h"):
        residual_norm.backward(None, None, (x, x), st)


@pytest.mark.parametrize("which", ["grad_r", "grad_h"])
def test_gradients_that_are_not_on_a_gpu(which):
    from actnn_b200.cpp_extension import residual_norm
    x, st = torch.zeros(4, 16), torch.zeros(4, 4)
    grads = (x, None) if which == "grad_r" else (None, x)
    with pytest.raises(RuntimeError, match="%s must be a CUDA tensor" % which):
        residual_norm.backward(*grads, (x, x), st)
