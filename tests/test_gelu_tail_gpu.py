"""GELU (erf) of 16-bit types far below zero: the values and slopes keep the digits of their type, where half of the distribution less
half of it would leave none."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# The normal distribution's tail: the polynomial of the fast form is off by 0.0103 of the tail at most down to -8
# (0.0016 down to -5), the slope with it by 2e-4; the hardware's exponential and reciprocal add 2e-5 of the value.
TAIL, SLOPE = 0.0104, 3e-4
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -130}     # half of the least step, generously


def exact(z):
    tail = 0.5 * torch.erfc(-z / math.sqrt(2.0))
    return z * tail, tail + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


@pytest.mark.parametrize("dtype", list(UNIT))
def test_values(cuda_device, dtype):
    from actnn_b200.cpp_extension import checkpoint
    x = torch.linspace(-8, -1, 5000, device="cuda").to(dtype)
    want = exact(x.double())[0]
    got = checkpoint.activation_forward(x, "gelu", save=False)[0]
    assert bool(((got.double() - want).abs() <= (TAIL + UNIT[dtype]) * want.abs() + LEAST[dtype]).all())


@pytest.mark.parametrize("dtype", list(UNIT))
def test_slopes(cuda_device, dtype):
    """Below -1, away from the slope's zero at -0.75."""
    from actnn_b200.cpp_extension import checkpoint
    x = torch.linspace(-8, -1, 5000, device="cuda").to(dtype)
    want = exact(x.double())[1]
    got = checkpoint.activation_backward(torch.ones_like(x), "gelu", x=x)
    assert bool(((got.double() - want).abs() <= (SLOPE + UNIT[dtype]) * want.abs() + LEAST[dtype]).all())


@pytest.mark.parametrize("dtype", list(UNIT))
def test_gated(cuda_device, dtype):
    """The gated form, by vectors and by single elements, times one: the same values."""
    from actnn_b200.cpp_extension import checkpoint
    x = torch.linspace(-8, 8, 4096, device="cuda").to(dtype)
    y = checkpoint.activation_forward(x, "gelu", save=False)[0]
    both = torch.stack([x, torch.ones_like(x)])
    assert torch.equal(checkpoint.activation_forward(both.t().contiguous().view(-1, 2), "gelu", gated=True, save=False)[0].view(-1), y)
    assert torch.equal(checkpoint.activation_forward(both.view(1, -1), "gelu", gated=True, save=False)[0].view(-1), y)
