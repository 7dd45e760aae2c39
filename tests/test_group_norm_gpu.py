"""Group norm with an activation and an 8-bit checkpoint, against the formulas in 64 bits."""
import pytest
import torch

from test_act_checkpoint_gpu import slope, value

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
EPS = 1e-5
# statistics, the scaled and shifted input and the functions: relative errors of a few fp32 roundings each, of sums whose
# threads add at most some hundred terms one after another
OWN = 2.0 ** -16


def data(shape, dtype, seed=0, mean=0.5):
    g = torch.Generator().manual_seed(seed)
    c = shape[1]
    x = torch.randn(shape, generator=g)
    side = [1, c] + [1] * (len(shape) - 2)
    return (x * torch.exp(0.3 * torch.randn(side, generator=g)) + mean * torch.randn(side, generator=g)).to(dtype).cuda()


def parameters(c, seed=9):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.3 * torch.randn(c, generator=g)).cuda(), (0.3 * torch.randn(c, generator=g)).cuda()


def last(x):
    return x.to(memory_format=torch.channels_last) if x.dim() == 4 else x


def rows(x, groups):
    return x.reshape(x.shape[0], groups, -1)


def definition(x, groups):
    """What the codes of x stand for, one rounded fp32 operation after another, on the CPU."""
    r = rows(x.detach().cpu().float(), groups)
    hi, lo = r.amax(2, keepdim=True), r.amin(2, keepdim=True)
    mid, half = 0.5 * hi + 0.5 * lo, (0.5 * hi - 0.5 * lo).clamp_min(1e-30)
    codes = ((r - mid) * (half.reciprocal() * 127.0)).round()
    step = half * torch.tensor(1 / 127, dtype=torch.float32)
    return codes.view(x.shape).to(torch.int8), mid, half, (mid.double() + codes.double() * step.double()).view(x.shape).to(x.device)


def reference(x, seen, groups, weight, bias, name, dy, eps=EPS):
    """Output from x; gradients at the input `seen`; and how large what they are made of is."""
    r = rows(x.double(), groups)
    var, mean = torch.var_mean(r, 2, correction=0, keepdim=True)
    rstd = (var + eps).rsqrt()
    side = [1, x.shape[1]] + [1] * (x.dim() - 2)
    w, b = ((torch.ones(side, dtype=torch.float64, device=x.device) * v) if p is None else p.double().view(side)
            for p, v in ((weight, 1), (bias, 0)))
    z = ((r - mean) * rstd).view(x.shape) * w + b
    size = ((r.abs() + mean.abs()) * rstd).view(x.shape) * w.abs() + b.abs() + 1
    h = ((rows(seen, groups) - mean) * rstd).view(x.shape)
    dz = dy.double() * slope(name, h * w + b)
    dims = [i for i in range(x.dim()) if i != 1]
    dn = rows(dz * w, groups)
    hr = rows(h, groups)
    dx = (rstd * (dn - dn.mean(2, keepdim=True) - hr * (dn * hr).mean(2, keepdim=True))).view(x.shape)
    off = rows(dy.double().abs() * (2 + size), groups) * w.abs().amax()
    offx = (rstd * (off + off.mean(2, keepdim=True) + hr.abs() * (off * hr.abs()).mean(2, keepdim=True))).view(x.shape)
    grads = (dx, (dz * h).sum(dims), dz.sum(dims))
    sizes = (offx, (dy.double().abs() * (2 + size) * (1 + h.abs())).sum(dims), (dy.double().abs() * (2 + size)).sum(dims))
    return value(name, z), size, grads, sizes


def near(got, ref, size):
    bound = UNIT[got.dtype] * ref.abs() + OWN * size + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    return got.shape == ref.shape and bool(((got.double() - ref).abs() <= bound).all())


SHAPES = [((1, 8, 1, 1), 1), ((2, 64, 14, 14), 8), ((3, 6, 5, 7), 2), ((2, 192, 9, 11), 32), ((1, 36, 8, 8), 4), ((2, 320, 6, 5), 32),
          ((2, 33, 4, 9), 3), ((1, 7, 13, 13), 7), ((2, 32, 3, 3), 32), ((1, 4, 300, 200), 1), ((2, 4104, 3, 2), 27), ((1, 2080, 2, 2), 1),
          ((1, 262, 3, 3), 2), ((1, 517, 4, 3), 1), ((2, 4096, 2, 3), 1), ((5, 48), 6), ((3, 40, 17), 5), ((2, 16, 3, 4, 5), 4), ((300, 16, 2, 2), 4)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_forward_codes_and_backward(cuda_device, dtype, shape, groups):
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import group_norm
    name = ["silu", "none", "relu", "gelu", "gelu_tanh"][(shape[1] + len(shape)) % 5]
    x, dy = last(data(shape, dtype)), last(data(shape, dtype, 1, 0.0))
    w, b = parameters(shape[1])
    y, codes, stats = group_norm.forward(x, groups, w, b, EPS, name)
    ref, mid, half, seen = definition(x, groups)
    assert torch.equal(codes.movedim(-1, 1).cpu(), ref)
    assert torch.equal(stats[..., 2].cpu(), mid.squeeze(2)) and torch.equal(stats[..., 3].cpu(), half.squeeze(2))
    out, size, grads, sizes = reference(x, seen, groups, w, b, name, dy)
    assert near(y, out, size)
    assert torch.equal(group_norm.inference(x, groups, w, b, EPS, name), y)
    if name == "relu":                      # a value whose sign the rounding may decide is left out
        side = [1, shape[1]] + [1] * (len(shape) - 2)
        r = rows(x.double(), groups)
        var, mean = torch.var_mean(r, 2, correction=0, keepdim=True)
        z = ((rows(seen, groups) - mean) * (var + EPS).rsqrt()).view(shape) * w.double().view(side) + b.double().view(side)
        assert not bool((z.abs() < 1e-6).any())
    gx, gw, gb = group_norm.backward(dy, codes, stats, groups, w, b, name)
    for got, want, scale in zip((gx, gw, gb), grads, sizes):
        assert near(got, want, scale)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    ops.group_norm.apply(x, groups, w, b, EPS, name).backward(dy)
    assert torch.equal(x.grad, gx) and torch.equal(w.grad, gw) and torch.equal(b.grad, gb)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["silu", "gelu", "none"])
@pytest.mark.parametrize("shape,groups", [((2, 64, 14, 14), 8), ((3, 33, 5, 7), 3), ((1, 36, 9, 8), 4)])
def test_exact_level(cuda_device, dtype, name, shape, groups):
    """Without compression the backward pass reads the input itself."""
    import actnn_b200 as actnn
    actnn.set_optimization_level("L0")
    x, dy = last(data(shape, dtype)), last(data(shape, dtype, 1, 0.0))
    layer = actnn.QGroupNorm(groups, shape[1], EPS, activation=name).cuda()
    with torch.no_grad():
        w, b = parameters(shape[1])
        layer.weight.copy_(w), layer.bias.copy_(b)
    x.requires_grad_()
    y = layer(x)
    y.backward(dy)
    out, size, grads, sizes = reference(x.detach(), x.detach().double(), groups, w, b, name, dy)
    assert near(y.detach(), out, size)
    for got, want, scale in zip((x.grad, layer.weight.grad, layer.bias.grad), grads, sizes):
        assert near(got, want, scale)


def test_exact_level_against_differences(cuda_device):
    import actnn_b200 as actnn
    from actnn_b200 import ops
    actnn.set_optimization_level("L0")
    shape, groups = (2, 12, 5, 3), 3
    x, dy, v = last(data(shape, torch.float32)), last(data(shape, torch.float32, 1, 0.0)), data(shape, torch.float32, 2, 0.0).double()
    w, b = parameters(12)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    ops.group_norm.apply(x, groups, w, b, EPS, "silu").backward(dy)

    def loss(z, ww, bb):
        return (torch.nn.functional.silu(torch.nn.functional.group_norm(z, groups, ww, bb, EPS)) * dy.double()).sum()

    z, e = x.detach().double(), 1e-5
    wd, bd, vw = w.detach().double(), b.detach().double(), torch.linspace(-1, 1, 12, dtype=torch.float64, device="cuda")
    size = float(dy.double().abs().sum()) * 50           # of the loss's first three derivatives along v
    assert abs(float((loss(z + e * v, wd, bd) - loss(z - e * v, wd, bd)) / (2 * e) - (x.grad.double() * v).sum())) <= OWN * size
    assert abs(float((loss(z, wd + e * vw, bd) - loss(z, wd - e * vw, bd)) / (2 * e) - (w.grad.double() * vw).sum())) <= OWN * size
    assert abs(float((loss(z, wd, bd + e * vw) - loss(z, wd, bd - e * vw)) / (2 * e) - (b.grad.double() * vw).sum())) <= OWN * size


def test_a_mean_far_from_zero(cuda_device):
    """Sums of squares would lose the variance: 1 beside 3000."""
    from actnn_b200.cpp_extension import group_norm
    g = torch.Generator().manual_seed(0)
    x = last((3000 + torch.randn(2, 32, 40, 40, generator=g)).cuda())
    x[0, 0, 0, 0] = 3100                                 # the first element stands out
    y = group_norm.inference(x, 4)
    ref = torch.nn.functional.group_norm(x.double(), 4, eps=EPS)
    assert float((y.double() - ref).abs().max()) <= 3000 * 2.0 ** -22 + 1e-4


def test_constant_groups_and_values_that_are_not_finite(cuda_device):
    from actnn_b200.cpp_extension import group_norm
    x = last(data((3, 16, 6, 6), torch.bfloat16))
    x[0, :4] = 2.0
    x[1, 5, 2, 2] = float("nan")
    x[2, 9, 0, 0] = float("inf")
    w, b = parameters(16)
    y, codes, stats = group_norm.forward(x, 4, w, b, EPS, "silu")
    assert torch.allclose(y[0, :4].float(), torch.nn.functional.silu(b[:4]).view(4, 1, 1).expand(4, 6, 6), atol=5e-3)
    bad = torch.zeros(3, 16, dtype=torch.bool, device="cuda")
    bad[1, 4:8] = bad[2, 8:12] = True
    lost = y.isnan().all((2, 3))
    assert bool(lost[1, 4:8].all()) and bool(y[~bad].isfinite().all())
    dy = last(data((3, 16, 6, 6), torch.bfloat16, 1))
    gx, gw, gb = group_norm.backward(dy, codes, stats, 4, w, b, "silu")
    assert bool(gx[~bad].isfinite().all()) and bool(gx[bad].isnan().all()) and bool(gw[:4].isfinite().all())


def test_other_memory_orders(cuda_device):
    from actnn_b200.cpp_extension import group_norm
    base = data((4, 24, 10, 12), torch.float16)
    w, b = parameters(24)
    want = group_norm.forward(last(base), 6, w, b, EPS, "silu")
    dy = data((4, 24, 10, 12), torch.float16, 1, 0.0)
    grads = group_norm.backward(last(dy), want[1], want[2], 6, w, b, "silu")
    y, codes, stats = group_norm.forward(base, 6, w, b, EPS, "silu")                 # planes
    assert torch.equal(y, want[0]) and torch.equal(codes, want[1]) and y.is_contiguous(memory_format=torch.channels_last)
    for g, ref in zip(group_norm.backward(dy, codes, stats, 6, w, b, "silu"), grads):
        assert torch.equal(g, ref)
    wide = torch.randn(4, 10, 12, 40, device="cuda").half()
    wide[..., 3:27] = base.permute(0, 2, 3, 1)
    assert torch.equal(group_norm.inference(wide[..., 3:27].permute(0, 3, 1, 2), 6, w, b, EPS, "silu"), want[0])
    assert torch.equal(group_norm.inference(last(base)[::2], 6, w, b, EPS, "silu"), want[0][::2])
    shifted = torch.empty(base.numel() + 4, dtype=torch.float16, device="cuda")[4:].view(4, 10, 12, 24)
    shifted.copy_(base.permute(0, 2, 3, 1))
    ref, size, _, _ = reference(base, base.double(), 6, w, b, "silu", dy)               # narrower vectors add in another order
    assert near(group_norm.inference(shifted.permute(0, 3, 1, 2), 6, w, b, EPS, "silu"), ref, size)
    dy1 = torch.ones(1, 1, 1, 1, device="cuda").half().expand(4, 24, 10, 12)            # a broadcast gradient
    a = group_norm.backward(dy1, want[1], want[2], 6, w, b, "silu")
    c = group_norm.backward(last(dy1.contiguous()), want[1], want[2], 6, w, b, "silu")
    assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_samples_do_not_depend_on_their_neighbours(cuda_device):
    from actnn_b200.cpp_extension import group_norm
    x = last(data((37, 64, 20, 20), torch.bfloat16))
    y = group_norm.inference(x, 8, activation="silu")
    again = group_norm.inference(x, 8, activation="silu")
    assert torch.equal(y, again)
    one = torch.cat([group_norm.inference(x[i:i + 1], 8, activation="silu") for i in range(37)])
    assert float((one.float() - y.float()).abs().max()) <= 2.0 ** -6


@pytest.mark.parametrize("shape", [(0, 8, 4, 4), (2, 8, 0, 4)])
def test_empty(cuda_device, shape):
    from actnn_b200 import ops
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    w, b = (torch.ones(8, device="cuda", requires_grad=True) for _ in range(2))
    y = ops.group_norm.apply(x, 2, w, b, EPS, "silu")
    y.sum().backward()
    assert y.shape == x.shape == x.grad.shape and not w.grad.any() and not b.grad.any()


def test_without_parameters_and_half_parameters(cuda_device):
    from actnn_b200 import ops
    x, dy = last(data((2, 16, 5, 5), torch.float16)), last(data((2, 16, 5, 5), torch.float16, 1, 0.0))
    a, c = x.clone().requires_grad_(), x.clone().requires_grad_()
    ops.group_norm.apply(a, 4, None, None, EPS, "silu").backward(dy)
    one, zero = torch.ones(16, device="cuda").half().requires_grad_(), torch.zeros(16, device="cuda").half().requires_grad_()
    ops.group_norm.apply(c, 4, one, zero, EPS, "silu").backward(dy)
    assert torch.equal(a.grad, c.grad) and one.grad.dtype == zero.grad.dtype == torch.float16


def test_many_samples(cuda_device):
    """More samples than a grid's second dimension holds."""
    from actnn_b200 import ops
    x = data((70000, 16), torch.float16).requires_grad_()
    w, b = (p.requires_grad_() for p in parameters(16))
    y = ops.group_norm.apply(x, 2, w, b, EPS, "none")
    ref = torch.nn.functional.group_norm(x.detach().double(), 2, w.detach().double(), b.detach().double(), EPS)
    assert float((y.double() - ref).abs().max()) <= 2.0 ** -9 * float(ref.abs().max())
    dy = data((70000, 16), torch.float16, 1, 0.0)
    y.backward(dy)
    assert bool(((b.grad.double() - dy.double().sum(0)).abs() <= OWN * dy.double().abs().sum(0)).all())


def test_beyond_two_to_the_31(cuda_device):
    from actnn_b200.cpp_extension import group_norm
    n, c, s = 3, 64, (1 << 31) // (64 * 3) + 1000
    x = torch.zeros(n, s, c, dtype=torch.float16, device="cuda")
    x[2, -1000:] = torch.randn(1000, c, device="cuda").half()
    x[0, :10] = 1.0
    y, codes, stats = group_norm.forward(x.movedim(-1, 1), 8, activation="none")
    ref = x[2].view(s, 8, 8)[-1000:].double()
    count = s * 8
    mean, sq = ref.sum((0, 2)) / count, ref.square().sum((0, 2)) / count
    rstd = (sq - mean * mean + EPS).rsqrt()
    want = ((ref - mean[None, :, None]) * rstd[None, :, None]).view(1000, c)
    got = y.movedim(1, -1)[2, -1000:].double()
    assert float((got - want).abs().max()) <= 2.0 ** -10 * float(want.abs().max())
    dy = torch.zeros_like(x)
    dy[2, -1000:] = 1.0
    gx, gw, gb = group_norm.backward(dy.movedim(-1, 1), codes, stats, 8)
    assert bool((gb == 1000).all()) and bool(gx.movedim(1, -1)[2, -5:].isfinite().all()) and bool(codes[2, -1000:].any())


@pytest.mark.parametrize("level", ["L3", "L4", "swap"])
def test_layer_and_levels(cuda_device, level):
    import actnn_b200 as actnn
    actnn.set_optimization_level(level)
    layer = actnn.QGroupNorm(4, 32, activation="silu").cuda()
    stock = torch.nn.Sequential(torch.nn.GroupNorm(4, 32), torch.nn.SiLU()).cuda()
    x, dy = last(data((4, 32, 12, 12), torch.float32)), last(data((4, 32, 12, 12), torch.float32, 1, 0.0))
    a, c = x.clone().requires_grad_(), x.clone().requires_grad_()
    y = layer(a)
    y.backward(dy)
    z = stock(c)
    z.backward(dy)
    assert torch.allclose(y, z, atol=1e-5, rtol=1e-5)
    # the saved input is off by half a step of its group's range, some 1 / 254 of it
    assert float((a.grad - c.grad).abs().max()) <= 0.05 * float(dy.abs().max()) * 2
    with torch.no_grad():
        assert torch.equal(layer(x), y)


def test_graph_and_stream(cuda_device):
    from actnn_b200.cpp_extension import group_norm
    x = last(data((3, 32, 9, 9), torch.bfloat16))
    w, b = parameters(32)
    want = group_norm.forward(x, 4, w, b, EPS, "gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [group_norm.forward(x, 4, w, b, EPS, "gelu") for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for g in got for p, q in zip(g, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = group_norm.forward(x, 4, w, b, EPS, "gelu")
    x.copy_(last(data((3, 32, 9, 9), torch.bfloat16, 4)))
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(out, group_norm.forward(x, 4, w, b, EPS, "gelu")))


def test_refusals(cuda_device):
    import actnn_b200 as actnn
    from actnn_b200.cpp_extension import group_norm
    x = last(data((2, 16, 4, 4), torch.float16))
    w, b = parameters(16)
    y, codes, stats = group_norm.forward(x, 4, w, b)
    bad = [lambda: group_norm.inference(x, 5), lambda: group_norm.inference(x, 0), lambda: group_norm.inference(x, 4, w[:8]),
           lambda: group_norm.inference(x.cpu(), 4), lambda: group_norm.inference(x.double(), 4), lambda: group_norm.inference(x[0, 0, 0], 1),
           lambda: group_norm.inference(x, 4, activation="swish"), lambda: group_norm.inference(x, 4, eps=-1.0),
           lambda: group_norm.inference(x, 4, w.cpu()), lambda: group_norm.backward(y[:1], codes, stats, 4, w, b),
           lambda: group_norm.backward(y, codes, stats[:1], 4, w, b), lambda: group_norm.backward(y, codes.float(), stats, 4, w, b),
           lambda: group_norm.backward(y, codes, stats, 2, w, b), lambda: actnn.QGroupNorm(4, 16, activation="swish")]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
