"""The 8-bit integer product against the same product in 64 bits, its row codes against their definition, and its gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# rounding of a result to its type; the scales, the bias and the conversion of the sum are at most eight fp32 roundings
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
FP32 = 8 * 2.0 ** -24
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def definition(x):
    """Codes and scales, one rounded fp32 operation after another, on the CPU."""
    a = x.detach().cpu().float().abs().amax(-1, keepdim=True).clamp_min(1e-30)
    codes = (x.detach().cpu().float() * (a.reciprocal() * 127.0)).round()
    return codes.to(torch.int8), (a * torch.tensor(1 / 127, dtype=torch.float32)).squeeze(-1)


def tokens(t, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(t, k, generator=g) * torch.exp(torch.randn(t, 1, generator=g))).to(dtype).cuda()


def check_product(y, codes, scale, wcodes, wscale, bias):
    product = (codes.double() @ wcodes.double().t()) * scale.double()[:, None] * wscale.double()
    ref = product if bias is None else product + bias.double()
    bound = (UNIT[y.dtype] + FP32) * ref.abs() + FP32 * product.abs() + (2.0 ** -25 if y.dtype == torch.float16 else 0)
    assert y.shape == ref.shape and bool(((y.double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (3, 7), (5, 8), (2, 1024), (9, 1032), (4, 2049), (3, 8192), (2, 9001), (300, 40)])
def test_row_codes(cuda_device, dtype, rows, cols):
    from actnn_b200.cpp_extension import int8
    x = tokens(rows, cols, dtype)
    if rows > 2:
        x[1] = 0
    codes, scale = int8.quantize_rows(x)
    ref, rscale = definition(x)
    assert torch.equal(codes.cpu(), ref) and torch.equal(scale.cpu(), rscale)
    stored = codes.as_strided((rows, codes.stride(0)), (codes.stride(0), 1))
    assert codes.stride(0) % 16 == 0 and not stored[:, cols:].any()
    for out in DTYPES:
        back = int8.dequantize_rows(codes, scale, out)
        assert torch.equal(back, (codes.float() * scale[:, None]).to(out))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_other_strides(cuda_device, dtype):
    """A slice of columns, every other row, a shifted start, a transposed matrix, an expanded row, more dimensions."""
    from actnn_b200.cpp_extension import int8
    base = tokens(40, 96, dtype)
    for x in (base[:, 8:72], base[:, 3:50], base[::2], base[1:, 1:], base.t(), base[:1].expand(7, 96), base.view(4, 10, 96),
              base.view(4, 10, 96).transpose(0, 1)):
        codes, scale = int8.quantize_rows(x)
        ref, rscale = definition(x)
        assert torch.equal(codes.cpu(), ref) and torch.equal(scale.cpu(), rscale)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_rows_that_are_not_finite_stay_apart(cuda_device, bad):
    from actnn_b200.cpp_extension import int8
    x, w = tokens(6, 200, torch.bfloat16), tokens(50, 200, torch.bfloat16, 1)
    clean = int8.linear(x, *int8.quantize_rows(w))
    x[2, 77] = bad
    y = int8.linear(x, *int8.quantize_rows(w))
    assert y[2].isnan().all() and torch.equal(y[[0, 1, 3, 4, 5]], clean[[0, 1, 3, 4, 5]])
    w[4, 0] = bad
    y = int8.linear(x, *int8.quantize_rows(w))
    assert y[:, 4].isnan().all() and torch.equal(y[[0, 1, 3]][:, :4], clean[[0, 1, 3]][:, :4])


def test_tiny_and_huge_rows(cuda_device):
    from actnn_b200.cpp_extension import int8
    x = torch.ones(4, 32, device="cuda")
    x[0], x[1], x[2] = 1e-42, 3e38, 1e-31
    codes, scale = int8.quantize_rows(x)
    assert torch.equal(codes.cpu(), definition(x)[0]) and scale.isfinite().all()
    assert int(codes[0].abs().max()) == 0 and int(codes[1].min()) == 127


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,n,k", [(1, 1, 1), (1, 128, 128), (1, 1000, 2048), (2, 33, 500), (3, 260, 129), (4, 128, 4100), (5, 129, 16),
                                   (8, 4096, 96), (9, 300, 1001), (15, 64, 256), (16, 128, 127), (17, 129, 1025), (31, 500, 640),
                                   (64, 70, 4096), (100, 1000, 777), (129, 640, 130), (255, 256, 384), (256, 257, 385), (257, 127, 2000),
                                   (600, 1111, 300), (1025, 2000, 144)])
def test_product(cuda_device, dtype, t, n, k):
    from actnn_b200.cpp_extension import int8
    x, w = tokens(t, k, dtype), tokens(n, k, dtype, 1)
    bias = None if (t + n) % 3 == 0 else tokens(1, n, dtype, 2)[0]
    wcodes, wscale = int8.quantize_rows(w)
    codes, scale = int8.quantize_rows(x)
    y = int8.linear(x, wcodes, wscale, bias)
    assert y.dtype == dtype
    check_product(y, codes, scale, wcodes, wscale, bias)
    z = int8.matmul(codes, scale, wcodes, wscale, bias, dtype)
    check_product(z, codes, scale, wcodes, wscale, bias)


@pytest.mark.parametrize("t", [1, 7, 40, 300])
def test_the_largest_sums_do_not_wrap(cuda_device, t):
    from actnn_b200.cpp_extension import int8
    k = int8.MOST_K
    codes = torch.full((t, k), 127, dtype=torch.int8, device="cuda")
    weights = torch.full((130, k), -127, dtype=torch.int8, device="cuda")
    one, ones = torch.ones(t, device="cuda"), torch.ones(130, device="cuda")
    y = int8.matmul(codes, one, weights, ones, dtype=torch.float32)
    assert torch.equal(y.double(), torch.full((t, 130), -127 * 127 * k, dtype=torch.float64, device="cuda").float().double())
    x = torch.ones(t, k, device="cuda")
    assert torch.equal(int8.linear(x, weights, ones)[:, 0], y[:, 0] * (torch.tensor(1.0) * torch.tensor(1 / 127)).cuda())


def test_codes_of_any_layout(cuda_device):
    """Codes that do not start on 16 bytes, whose rows are not 16 bytes apart, or that run the other way are laid out anew."""
    from actnn_b200.cpp_extension import int8
    g = torch.Generator().manual_seed(3)
    base = torch.randint(-127, 128, (60, 101), generator=g).to(torch.int8).cuda()
    scale = torch.rand(60, generator=g).cuda() + 0.1
    for c, s in ((base, scale), (base[1:, 3:90], scale[1:]), (base[::2], scale[::2]), (base.t()[:50], torch.rand(50, device="cuda"))):
        for t in (3, 20):
            x = torch.randint(-127, 128, (t, c.shape[1]), generator=g).to(torch.int8).cuda()
            xs = torch.rand(t, generator=g).cuda()
            check_product(int8.matmul(x, xs, c, s, dtype=torch.bfloat16), x, xs, c, s, None)


def test_what_lies_behind_the_rows_is_not_read_as_data(cuda_device):
    from actnn_b200.cpp_extension import int8
    for t in (2, 30):
        codes, weights = (torch.full((r, 112), 99, dtype=torch.int8, device="cuda") for r in (t, 40))
        codes[:, :100] = 1
        weights[:, :100] = 2
        y = int8.matmul(codes[:, :100], torch.ones(t, device="cuda"), weights[:, :100], torch.ones(40, device="cuda"), dtype=torch.float32)
        assert bool((y == 200).all())
        x = torch.zeros(t, 100, device="cuda")
        x[:, 0] = 1
        y = int8.linear(x, weights[:, :100], torch.ones(40, device="cuda"))
        assert bool((y == 2 * (127 * torch.tensor(1 / 127)).cuda()).all())


@pytest.mark.parametrize("shape", [(0, 5, 16), (5, 0, 16), (4, 6, 0), (0, 0, 0)])
def test_empty(cuda_device, shape):
    from actnn_b200.cpp_extension import int8
    t, n, k = shape
    x, w, b = torch.randn(t, k, device="cuda"), torch.randn(n, k, device="cuda"), torch.randn(n, device="cuda")
    y = int8.linear(x, *int8.quantize_rows(w), b)
    assert y.shape == (t, n) and (k > 0 or torch.equal(y, b.expand(t, n)))


def test_more_dimensions_and_one(cuda_device):
    from actnn_b200.cpp_extension import int8
    x, w = tokens(24, 80, torch.float16), tokens(30, 80, torch.float16, 1)
    code = int8.quantize_rows(w)
    y = int8.linear(x, *code)
    assert torch.equal(int8.linear(x.view(2, 3, 4, 80), *code), y.view(2, 3, 4, 30))
    one = int8.linear(x[5], *code)
    assert one.shape == (30,) and torch.equal(one, int8.linear(x[5:6], *code)[0])


def test_another_stream(cuda_device):
    from actnn_b200.cpp_extension import int8
    x, w = tokens(70, 512, torch.bfloat16), tokens(300, 512, torch.bfloat16, 1)
    code = int8.quantize_rows(w)
    want = [int8.linear(x[:t], *code) for t in (1, 70)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [int8.linear(x[:t], *code) for t in (1, 70) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, want[i // 3]) for i, g in enumerate(got))


@pytest.mark.parametrize("t", [2, 48])
def test_a_captured_graph_replays(cuda_device, t):
    from actnn_b200.cpp_extension import int8
    x, w = tokens(t, 256, torch.bfloat16), tokens(200, 256, torch.bfloat16, 1)
    code = int8.quantize_rows(w)
    int8.linear(x, *code)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = int8.linear(x, *code)
    x.copy_(tokens(t, 256, torch.bfloat16, 9))
    graph.replay()
    assert torch.equal(y, int8.linear(x, *code))


def test_outputs_beyond_two_gigabytes(cuda_device):
    """Offsets of the output pass 31 bits of elements."""
    from actnn_b200.cpp_extension import int8
    t, n = 70001, 32768
    codes = torch.ones(t, 16, dtype=torch.int8, device="cuda")
    weights = torch.ones(n, 16, dtype=torch.int8, device="cuda")
    scale = (torch.arange(t, device="cuda") % 128).float()
    y = int8.matmul(codes, scale, weights, torch.ones(n, device="cuda"), dtype=torch.float16)
    assert bool((y[-300:].float() == (16 * scale[-300:, None])).all()) and bool((y[:, -1].float() == 16 * scale).all())
    assert bool((y[:, 0].float() == 16 * scale).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,n,with_bias", [((5, 24), 7, True), ((3, 4, 130), 65, False), ((200, 64), 129, True)])
def test_gradients(cuda_device, dtype, shape, n, with_bias):
    """Those of the product of the decoded matrices: dx = dy w^, dw = dy^T x^, db = sum of dy."""
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import int8
    k = shape[-1]
    rows = torch.Size(shape[:-1]).numel()
    x, w = tokens(rows, k, dtype).view(shape).requires_grad_(), tokens(n, k, dtype, 1).requires_grad_()
    b = tokens(1, n, dtype, 2)[0].requires_grad_() if with_bias else None
    y = ops.int8_linear.apply(x, w, b)
    dy = tokens(rows, n, dtype, 3).view(y.shape)
    y.backward(dy)
    xq = int8.dequantize_rows(*int8.quantize_rows(x.detach().view(-1, k)), torch.float32).double()
    wq = int8.dequantize_rows(*int8.quantize_rows(w.detach()), torch.float32).double()
    g = dy.double().view(-1, n)
    # operands decoded to the type (one rounding each), sums in fp32 over `terms`, the result rounded
    u = UNIT[dtype]
    for got, ref, size, terms in ((x.grad, g @ wq, g.abs() @ wq.abs(), n), (w.grad, g.t() @ xq, g.t().abs() @ xq.abs(), rows)):
        bound = (u + (terms + 8) * 2.0 ** -24) * size + u * ref.abs()
        assert got.dtype == dtype and bool(((got.double().view(ref.shape) - ref).abs() <= bound).all())
    if with_bias:
        bound = (rows + 8) * 2.0 ** -24 * g.abs().sum(0) + u * g.sum(0).abs() + u * g.abs().amax(0)
        assert bool(((b.grad.double() - g.sum(0)).abs() <= bound).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(0, 5), (1, 1), (3, 0), (31, 64), (33, 65), (700, 1000), (5000, 8), (64, 4104), (2, 20000)])
def test_column_sums(cuda_device, dtype, rows, cols):
    from actnn_b200.cpp_extension import int8
    x = tokens(rows, cols, dtype)
    got, ref = int8.column_sums(x), x.double().sum(0)
    bound = UNIT[dtype] * ref.abs() + (rows + 8) * 2.0 ** -24 * x.double().abs().sum(0) + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert got.dtype == dtype and got.shape == (cols,) and bool(((got.double() - ref).abs() <= bound).all())
    if rows > 2:
        y = torch.cat([x, x], 1)[:, cols // 2:cols // 2 + cols]                      # strides and starts that no vector fits
        assert torch.equal(int8.column_sums(y), int8.column_sums(y.contiguous()))


def test_gradients_against_differences(cuda_device):
    """Along a direction that keeps every code (one common factor), the loss moves as the gradient says."""
    from actnn_b200 import ops
    x, w = tokens(9, 33, torch.float32).requires_grad_(), tokens(12, 33, torch.float32, 1).requires_grad_()
    b, dy = tokens(1, 12, torch.float32, 2)[0].requires_grad_(), tokens(9, 12, torch.float32, 3)

    def loss(f, h):
        return float((ops.int8_linear.apply(x.detach() * f, w.detach() * h, b.detach()).double() * dy.double()).sum())

    (ops.int8_linear.apply(x, w, b) * dy).sum().backward()
    from actnn_b200.cpp_extension import int8
    xq = int8.dequantize_rows(*int8.quantize_rows(x.detach()), torch.float32)
    wq = int8.dequantize_rows(*int8.quantize_rows(w.detach()), torch.float32)
    size = float((xq.abs() @ wq.abs().t() * dy.abs()).sum())
    # the product is linear in each factor, powers of two keep every code: a difference is exact up to the fp32 sums
    assert abs((loss(2, 1) - loss(1, 1)) - float((x.grad.double() * xq.double()).sum())) <= 64 * 2.0 ** -24 * size
    assert abs((loss(1, 2) - loss(1, 1)) - float((w.grad.double() * wq.double()).sum())) <= 64 * 2.0 ** -24 * size


def test_gradients_that_are_not_asked_for(cuda_device):
    from actnn_b200 import ops
    x, w, b = tokens(4, 16, torch.float32), tokens(3, 16, torch.float32, 1), tokens(1, 3, torch.float32, 2)[0]
    for flags in ((True, False, False), (False, True, False), (False, False, True)):
        p = [v.clone().requires_grad_(f) for v, f in zip((x, w, b), flags)]
        ops.int8_linear.apply(*p).sum().backward()
        assert [v.grad is not None for v in p] == list(flags)


@pytest.mark.parametrize("level", ["L3", "swap", "L4"])
def test_layer_in_training_and_frozen(cuda_device, level):
    import actnn_b200 as actnn
    actnn.set_optimization_level(level)
    layer = actnn.QInt8Linear(96, 50).cuda().half()
    x = tokens(12, 96, torch.float16).requires_grad_()
    y = layer(x)
    y.sum().backward()
    assert x.grad.isfinite().all() and layer.weight.grad.shape == layer.weight.shape and layer.bias.grad.shape == (50,)
    layer.eval().freeze()
    with torch.no_grad():
        assert torch.equal(layer(x), y)
        layer.weight.zero_()
        assert torch.equal(layer(x), y)                   # the codes, until they are given up
        assert bool((layer.unfreeze()(x) == layer.bias).all())
    with pytest.raises(RuntimeError, match="frozen"):
        layer.freeze()(x)
    layer.train()
    assert layer.frozen is None


def test_under_autocast(cuda_device):
    import actnn_b200 as actnn
    layer = actnn.QInt8Linear(64, 32).cuda()
    x = tokens(10, 64, torch.float32).requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layer(x)
    assert y.dtype == torch.bfloat16
    y.float().square().sum().backward()
    assert x.grad.dtype == torch.float32 and layer.weight.grad.dtype == torch.float32 and layer.bias.grad.dtype == torch.float32


def test_refusals(cuda_device):
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import int8
    x, w = tokens(4, 32, torch.float16), tokens(6, 32, torch.float16, 1)
    codes, scale = int8.quantize_rows(w)
    xc, xs = int8.quantize_rows(x)
    bad = [lambda: int8.linear(x[:, :31], codes, scale), lambda: int8.linear(x.cpu(), codes, scale),
           lambda: int8.linear(x.double(), codes, scale), lambda: int8.linear(x, codes.float(), scale),
           lambda: int8.linear(x, codes, scale.half()), lambda: int8.linear(x, codes, scale[:5]),
           lambda: int8.linear(x, codes, scale, torch.zeros(5, device="cuda")), lambda: int8.linear(x, codes.cpu(), scale.cpu()),
           lambda: int8.matmul(xc, xs, codes, scale, dtype=torch.float64), lambda: int8.matmul(xc, xs[:2], codes, scale),
           lambda: int8.quantize_rows(torch.tensor(1.0, device="cuda")), lambda: int8.quantize_rows(x.int()),
           lambda: ops.int8_linear.apply(x, w[:, :30], None),
           lambda: int8.matmul(torch.zeros(1, int8.MOST_K + 1, dtype=torch.int8, device="cuda"), xs[:1],
                               torch.zeros(1, int8.MOST_K + 1, dtype=torch.int8, device="cuda"), scale[:1])]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    check_product(int8.linear(x, codes, scale), xc, xs, codes, scale, None)       # and nothing is left behind
