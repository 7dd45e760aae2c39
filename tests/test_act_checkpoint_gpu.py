"""Activation functions with an 8-bit checkpoint, against the formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# what the functions themselves are off before the rounding, relative and absolute (per unit of |z| or of what multiplies
# them): expf, erff and a rounded division within 4 ulp each for float32; exponential and reciprocal of the hardware for the
# 16-bit types, whose argument up to 30 carries a relative 2^-24 into the exponent
OWN = {torch.float32: 2.0 ** -20, torch.float16: 2.0 ** -17, torch.bfloat16: 2.0 ** -17}
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
KINDS = ["none", "relu", "silu", "gelu", "gelu_tanh"]
LEAST = 2.0 ** -25                      # half the spacing of the smallest float16 numbers


def value(name, z):
    if name == "relu":
        return z.clamp(min=0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def slope(name, z):
    z = z.detach().clone().requires_grad_()
    return torch.autograd.grad(value(name, z).sum(), z)[0] if name != "relu" else (z > 0).double()


def blocks_of(x):
    flat = x.reshape(-1)
    return torch.cat([flat, flat.new_zeros(-flat.numel() % 256)]).view(-1, 256)


def definition(x):
    """Codes and scales of 256 consecutive elements, one rounded fp32 operation after another, on the CPU."""
    b = blocks_of(x.detach().cpu().float())
    a = b.abs().amax(1, keepdim=True).clamp_min(1e-30)
    return (b * (a.reciprocal() * 127.0)).round().to(torch.int8), (a * torch.tensor(1 / 127, dtype=torch.float32)).squeeze(1)


def decoded(x):
    codes, scale = definition(x)
    return (codes.double() * scale.double()[:, None]).reshape(-1)[:x.numel()].view(x.shape).to(x.device)


def data(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (2.5 * torch.randn(shape, generator=g)).to(dtype).cuda()


def close(got, ref, scale):
    """One rounding of the result, and the functions' own error times what multiplies them."""
    bound = UNIT[got.dtype] * ref.abs() + OWN[got.dtype] * scale + (LEAST if got.dtype == torch.float16 else 0)
    return got.shape == ref.shape and bool(((got.double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", KINDS)
@pytest.mark.parametrize("shape", [(1,), (7,), (255,), (256,), (257,), (3, 1001), (64, 256), (5, 7, 130), (2, 4096)])
def test_activation(cuda_device, dtype, name, shape):
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import checkpoint
    x, dy = data(shape, dtype), data(shape, dtype, 1)
    y, codes, scale = checkpoint.activation_forward(x, name)
    ref, rscale = definition(x)
    assert torch.equal(codes.cpu().view(-1, 256), ref) and torch.equal(scale.cpu(), rscale)
    z = x.double()
    assert close(y, value(name, z), 1 + z.abs())
    z = decoded(x)
    dx = checkpoint.activation_backward(dy, name, codes, scale)
    assert close(dx, dy.double() * slope(name, z), dy.double().abs() * (2 + z.abs()))
    x.requires_grad_()
    ops.activation.apply(x, name).backward(dy)
    assert torch.equal(x.grad, dx)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", KINDS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 5), (1, 256), (7, 24), (9, 100), (5, 129), (33, 1000), (2, 4097), (300, 33)])
def test_gated(cuda_device, dtype, name, rows, cols):
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import checkpoint
    x, dy = data((rows, 2 * cols), dtype), data((rows, cols), dtype, 1)
    y, codes, scale = checkpoint.activation_forward(x, name, gated=True)
    gate, up = x[:, :cols], x[:, cols:]
    for half, part in enumerate((gate, up)):
        ref, rscale = definition(part.contiguous())
        assert torch.equal(codes.cpu().view(2, -1, 256)[half], ref) and torch.equal(scale.cpu().view(2, -1)[half], rscale)
    g, u = gate.double(), up.double()
    assert close(y, value(name, g) * u, (1 + g.abs()) * u.abs())
    g, u, d = decoded(gate.contiguous()), decoded(up.contiguous()), dy.double()
    dx = checkpoint.activation_backward(dy, name, codes, scale, gated=True)
    assert close(dx[:, :cols], d * u * slope(name, g), (d * u).abs() * (2 + g.abs()))
    assert close(dx[:, cols:], d * value(name, g), d.abs() * (1 + g.abs()))
    x.requires_grad_()
    ops.glu.apply(x, name).backward(dy)
    assert torch.equal(x.grad, dx)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh"])
def test_exact_level_against_differences(cuda_device, name, gated):
    """Without compression the backward pass reads the input: central differences of the forward pass in 64 bits."""
    import actnn_b200 as actnn
    from actnn_b200 import ops
    actnn.set_optimization_level("L0")
    x, dy = data((6, 36), torch.float32).requires_grad_(), data((6, 18 if gated else 36), torch.float32, 1)
    (ops.glu if gated else ops.activation).apply(x, name).backward(dy)
    v, e = data((6, 36), torch.float32, 2).double(), 1e-5

    def loss(z):
        y = value(name, z[:, :18]) * z[:, 18:] if gated else value(name, z)
        return (y * dy.double()).sum()

    z = x.detach().double()
    change = (loss(z + e * v) - loss(z - e * v)) / (2 * e)
    # the difference quotient: third derivatives below 30 here, e^2 of them, and 2^-52 / e of the loss's terms
    terms = float((dy.double().abs().sum() * 30 * (1 + v.abs().max()) ** 3))
    assert abs(float(change - (x.grad.double() * v).sum())) <= terms * e * e + 1e-9 * terms + OWN[torch.float32] * terms


@pytest.mark.parametrize("gated,cols", [(False, 40), (True, 40), (True, 37)])
def test_blocks_of_zeros_and_values_that_are_not_finite(cuda_device, gated, cols):
    from actnn_b200.cpp_extension import checkpoint
    rows = 64
    x, dy = data((rows, cols * (2 if gated else 1)), torch.bfloat16), data((rows, cols), torch.bfloat16, 1)
    x[:32] = 0
    x[40, 3] = float("nan")
    x[50, 5] = float("inf")
    y, codes, scale = checkpoint.activation_forward(x, "gelu", gated=gated)
    dx = checkpoint.activation_backward(dy, "gelu", codes, scale, gated=gated)
    assert not y[:32].any() and y[40, 3].isnan() and bool(y[33:40].isfinite().all())
    first = [(r * cols + c) // 256 for r, c in ((40, 3), (50, 5))]           # whole blocks are lost, and no others
    block = torch.arange(rows * cols, device="cuda").view(rows, cols) // 256
    lost = (block == first[0]) | (block == first[1])
    part = dx[:, :cols]
    assert bool(part[~lost].isfinite().all()) and bool(part[lost].isnan().all())


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("name", KINDS[1:])
def test_far_out(cuda_device, name, gated):
    """Arguments whose squares and exponentials overflow."""
    from actnn_b200.cpp_extension import checkpoint
    z = torch.tensor([1e30, -1e30, 3e19, -3e19, 200., -200., 90., -90., 0., 40., -40., 88.], device="cuda")
    x = torch.cat([z, torch.ones_like(z)]).view(1, -1) if gated else z.view(1, -1)
    y = checkpoint.activation_forward(x, name, gated=gated)[0]
    dx = checkpoint.activation_backward(torch.ones_like(y), name, x=x, gated=gated)[:, :12]
    ref, dref = value(name, z.double().clamp(min=-1e3)), slope(name, z.double().clamp(-1e3, 1e3))
    ref = torch.where(z < -1e3, 0., ref)
    assert bool(((y.double() - ref).abs() <= 1e-6 * ref.abs() + 1e-30).all())
    assert bool(((dx.double() - dref).abs() <= 1e-5).all())


@pytest.mark.parametrize("gated", [False, True])
def test_other_strides_and_starts(cuda_device, gated):
    from actnn_b200.cpp_extension import checkpoint
    base = data((40, 200), torch.float16)
    for x in (base[:, 8:104], base[::3], base.t(), base.reshape(-1)[1:4001].view(20, 200), base.reshape(-1)[4:4004].view(20, 200),
              base[:1].expand(6, 200)):
        y, codes, scale = checkpoint.activation_forward(x, "silu", gated=gated)
        want = checkpoint.activation_forward(x.contiguous().clone(), "silu", gated=gated)
        assert torch.equal(y, want[0]) and torch.equal(codes, want[1]) and torch.equal(scale, want[2])
        dy = data((y.shape[1], y.shape[0]), torch.float16, 1).t()
        assert torch.equal(checkpoint.activation_backward(dy, "silu", codes, scale, gated=gated),
                           checkpoint.activation_backward(dy.contiguous(), "silu", codes, scale, gated=gated))


@pytest.mark.parametrize("shape", [(0,), (0, 8), (4, 0), ()])
def test_empty_and_scalars(cuda_device, shape):
    from actnn_b200 import ops
    x = torch.full(shape, 0.5, device="cuda", requires_grad=True)
    ops.activation.apply(x, "silu").sum().backward()
    assert x.grad.shape == x.shape
    if len(shape) == 2:
        y = ops.glu.apply(torch.zeros(shape[0], 2 * shape[1], device="cuda", requires_grad=True), "silu")
        assert y.shape == shape
        y.sum().backward()


@pytest.mark.parametrize("gated,cols", [(False, 4096), (True, 4096), (True, 4095)])
def test_beyond_two_to_the_31(cuda_device, gated, cols):
    """Offsets of inputs and codes pass 31 bits."""
    from actnn_b200.cpp_extension import checkpoint
    rows = (1 << 31) // (cols * (2 if gated else 1)) + 3
    x = torch.zeros(rows, cols * (2 if gated else 1), dtype=torch.float16, device="cuda")
    x[-4:] = data((4, x.shape[1]), torch.float16)
    y, codes, scale = checkpoint.activation_forward(x, "silu", gated=gated)
    tail = value("silu", x[-4:, :cols].double()) * (x[-4:, cols:].double() if gated else 1)
    assert close(y[-4:], tail, 30 + tail.abs()) and not y[:-4].any()
    dx = checkpoint.activation_backward(torch.ones_like(y), "silu", codes, scale, gated=gated)
    z = x[-3:, :cols].double()
    near = slope("silu", z) * (x[-3:, cols:].double() if gated else 1)
    assert bool(((dx[-3:, :cols].double() - near).abs() <= 0.25).all()) and dx.shape == x.shape


def test_layers_and_levels(cuda_device):
    import actnn_b200 as actnn
    x, dy = data((10, 64), torch.float16), data((10, 64), torch.float16, 1)
    grads = {}
    for level in ("L3", "L4", "L0", "swap"):
        actnn.config.__dict__.update(actnn.conf.QuantizationConfig().__dict__)
        actnn.set_optimization_level(level)
        for layer, stock in ((actnn.QSiLU(), torch.nn.SiLU()), (actnn.QGELU(), torch.nn.GELU()),
                             (actnn.QGELU("tanh"), torch.nn.GELU("tanh"))):
            a, b = (x.clone().requires_grad_() for _ in range(2))
            layer(a).backward(dy)
            stock(b).backward(dy)
            step = float(x.abs().max()) / 127
            assert float((a.grad - b.grad).abs().max()) <= (step if level in ("L3", "L4") else 0.01) * float(dy.abs().max())
            grads.setdefault(layer.extra_repr(), []).append(a.grad)
            with torch.no_grad():
                assert torch.equal(layer(x), layer(a).detach())
    for g in grads.values():
        assert torch.equal(g[0], g[1]) and torch.equal(g[2], g[3])
    with torch.no_grad():
        gate, up = x.chunk(2, -1)
        assert torch.allclose(actnn.QGLU("silu")(x).float(), torch.nn.functional.silu(gate).float() * up.float(), atol=1e-2, rtol=2e-3)


def test_graph_and_stream(cuda_device):
    from actnn_b200.cpp_extension import checkpoint
    x = data((30, 512), torch.bfloat16)
    want = checkpoint.activation_forward(x, "gelu", gated=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = checkpoint.activation_forward(x, "gelu", gated=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = checkpoint.activation_forward(x, "gelu", gated=True)
    x.copy_(data((30, 512), torch.bfloat16, 5))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, checkpoint.activation_forward(x, "gelu", gated=True)))


def test_refusals(cuda_device):
    import actnn_b200 as actnn
    from actnn_b200.cpp_extension import checkpoint
    x = data((4, 64), torch.float16)
    y, codes, scale = checkpoint.activation_forward(x, "silu")
    bad = [lambda: checkpoint.activation_forward(x, "tanh"), lambda: checkpoint.activation_forward(x.cpu(), "silu"),
           lambda: checkpoint.activation_forward(x.double(), "silu"), lambda: checkpoint.activation_forward(x[:, :63], "silu", gated=True),
           lambda: checkpoint.activation_backward(y, "silu", codes[:-256], scale), lambda: checkpoint.activation_backward(y, "silu", codes, None),
           lambda: checkpoint.activation_backward(y, "silu", codes.float(), scale), lambda: checkpoint.activation_backward(y, "silu"),
           lambda: checkpoint.activation_backward(y, "silu", x=x[:2]), lambda: checkpoint.activation_backward(y, "silu", codes, scale, gated=True),
           lambda: checkpoint.activation_backward(y, "silu", codes.cpu(), scale.cpu()), lambda: actnn.QGLU("swish")]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        actnn.QGELU("erf")
