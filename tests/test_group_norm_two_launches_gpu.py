"""Group norm on tensors that its two launches each way take: rings of copies that wrap, partial results that are folded between
the launches, vectors whose channels are of two or three groups."""
import pytest
import torch

from test_group_norm_gpu import DTYPES, EPS, definition, near, parameters, reference

pytestmark = pytest.mark.gpu

SHAPES = [((130, 256, 28, 20), 32),        # a few runs of positions a sample, some thirty a thread
          ((6, 256, 100, 90), 32),         # many runs: folded
          ((100, 192, 35, 35), 32),        # six channels a group
          ((20, 96, 64, 63), 16),          # six channels a group, folded
          ((40, 192, 30, 31), 64),         # three channels a group: a vector of eight touches four groups
          ((12, 4096, 21, 19), 1),         # a group wider than a block: parts of it, folded
          ((24, 36, 70, 70), 6),           # vectors of four
          ((150, 34, 41, 40), 2),          # of two
          ((60, 33, 50, 41), 3),           # single elements
          ((3, 512, 128, 127), 512)]       # an instance norm: tables of 256 groups a block


def on_device(shape, dtype, seed, mean):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, c = shape[:2]
    x = torch.randn((n,) + tuple(shape[2:]) + (c,), generator=g, device="cuda")
    x.mul_(torch.exp(0.3 * torch.randn(c, generator=g, device="cuda"))).add_(mean * torch.randn(c, generator=g, device="cuda"))
    return x.to(dtype).movedim(-1, 1)                    # channels last


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_forward_codes_and_backward(cuda_device, dtype, shape, groups):
    from actnn_b200.cpp_extension import group_norm
    name = ["silu", "none", "gelu", "gelu_tanh"][(shape[0] + shape[1]) % 4]
    x, dy = on_device(shape, dtype, 0, 0.5), on_device(shape, dtype, 1, 0.0)
    w, b = parameters(shape[1])
    y, codes, stats = group_norm.forward(x, groups, w, b, EPS, name)
    ref, mid, half, seen = definition(x, groups)
    assert torch.equal(codes.movedim(-1, 1).cpu(), ref)
    assert torch.equal(stats[..., 2].cpu(), mid.squeeze(2)) and torch.equal(stats[..., 3].cpu(), half.squeeze(2))
    out, size, grads, sizes = reference(x, seen, groups, w, b, name, dy)
    assert near(y, out, size)
    assert torch.equal(group_norm.inference(x, groups, w, b, EPS, name), y)
    first = group_norm.backward(dy, codes, stats, groups, w, b, name)
    for got, want, scale in zip(first, grads, sizes):
        assert near(got, want, scale)
    for got, want in zip(group_norm.backward(dy, codes, stats, groups, w, b, name), first):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,groups", SHAPES[:4])
def test_the_input_itself_kept(cuda_device, dtype, shape, groups):
    from actnn_b200.cpp_extension import group_norm
    x, dy = on_device(shape, dtype, 2, 0.5), on_device(shape, dtype, 3, 0.0)
    w, b = parameters(shape[1])
    y, saved, stats = group_norm.forward(x, groups, w, b, EPS, "silu", compress=False)
    out, size, grads, sizes = reference(x, x.double(), groups, w, b, "silu", dy)
    assert near(y, out, size)
    for got, want, scale in zip(group_norm.backward(dy, saved, stats, groups, w, b, "silu"), grads, sizes):
        assert near(got, want, scale)
