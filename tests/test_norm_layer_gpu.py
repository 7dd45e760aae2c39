"""QGroupNorm gives every parameter that is trained its gradient, whatever else is."""
import itertools

import pytest
import torch

from test_group_norm_gpu import EPS, data, parameters

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("level", ["L3", "L0", "L4"])
@pytest.mark.parametrize("flags", list(itertools.product([False, True], repeat=3)))
def test_gradients_for_what_asks_for_one(cuda_device, flags, level):
    import actnn_b200 as actnn
    from actnn_b200 import ops
    actnn.set_optimization_level(level)
    x, dy = data((3, 24, 5, 7), torch.float32), data((3, 24, 5, 7), torch.float32, 1, 0.0)
    w, b = parameters(24)
    every = [v.clone().requires_grad_() for v in (x, w, b)]
    ops.group_norm.apply(every[0], 4, every[1], every[2], EPS, "silu").backward(dy)
    layer = actnn.QGroupNorm(4, 24, EPS, activation="silu").cuda()
    with torch.no_grad():
        layer.weight.copy_(w), layer.bias.copy_(b)
    mine = (x.clone().requires_grad_(flags[0]), layer.weight.requires_grad_(flags[1]), layer.bias.requires_grad_(flags[2]))
    y = layer(mine[0])
    assert y.requires_grad == any(flags)
    if any(flags):
        y.backward(dy)
    for got, want, asked in zip(mine, every, flags):
        assert torch.equal(got.grad, want.grad) if asked else got.grad is None
    with torch.no_grad():
        assert torch.equal(layer(mine[0]), y)
