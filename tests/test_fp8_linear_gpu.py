"""The 8-bit floating-point codes against their definition, their product against the same product in 64 bits, and its gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
CODES = torch.float8_e4m3fn


def two(e):
    """2^e in 64 bits, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def definition(x, high, wide):
    """What the codes of blocks of high x wide stand for, in 64 bits on the CPU, and the blocks' exponents."""
    x = x.detach().cpu().double()
    rows, cols = x.shape
    full = torch.nn.functional.pad(x, (0, -cols % wide, 0, -rows % high))
    tiles = full.view(full.shape[0] // high, high, -1, wide)
    a = torch.where(tiles.isfinite(), tiles.abs(), 0.0).amax((1, 3), keepdim=True)
    m, e = torch.frexp(a)
    e = torch.where(a > 0, (e - 9 + (m > 0.875).int()).clamp_min(-126), -126)
    code = torch.where(tiles.isfinite(), tiles * two(-e), float("nan")).float().to(CODES)
    return (code.double() * two(e)).view(full.shape)[:rows, :cols], e.view(e.shape[0], -1)


def same(a, b):
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def tokens(t, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(t, k, generator=g) * torch.exp(torch.randn(t, 1, generator=g)) / 16).to(dtype).cuda()


def decoded(codes, scales):
    from actnn_b200.cpp_extension import fp8
    return fp8.dequantize(codes, scales, torch.float32).double()


def check_product(y, x, w, bias=None):
    """x and w decoded, in 64 bits.  A product of codes is exact in fp32; a sum of K of them is off by at most 2^-23 of the magnitudes it
    passes through for each addition, rounded or cut off, and the bias adds one more."""
    ref, mag = x @ w.t(), x.abs() @ w.abs().t()
    bound = (x.shape[1] + 2) * 2.0 ** -23 * mag
    if bias is not None:
        ref = ref + bias.double()
        bound = bound + 2.0 ** -23 * bias.double().abs()
    bound = bound + UNIT[y.dtype] * (ref.abs() + bound) + (2.0 ** -25 if y.dtype == torch.float16 else 0)
    assert y.shape == ref.shape and bool(((y.double() - ref).abs() <= bound).all())


SHAPES = [(1, 1), (1, 16), (3, 7), (5, 8), (2, 127), (2, 128), (9, 129), (128, 128), (129, 257), (4, 511), (4, 512), (3, 513), (300, 40), (131, 1001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_codes(cuda_device, dtype, rows, cols):
    from actnn_b200.cpp_extension import fp8
    x = tokens(rows, cols, dtype)
    if rows > 2:
        x[1] = 0
    codes, scales = fp8.quantize(x)
    ref, e = definition(x, 1, 128)
    assert codes.dtype == CODES and torch.equal(decoded(codes, scales).cpu(), ref)
    blocks = scales.view(scales.shape[0], -1, 32, 4, 4).permute(1, 3, 2, 0, 4).reshape(-1, scales.shape[0] * 4)     # the order, undone
    assert torch.equal(blocks[:rows, :e.shape[1]].cpu().int(), e.int() + 127)
    raw = codes.view(torch.uint8)
    stored = raw.as_strided((rows, raw.stride(0)), (raw.stride(0), 1))
    assert raw.stride(0) % 16 == 0 and not stored[:, cols:].any()
    for out in DTYPES:
        assert same(fp8.dequantize(codes, scales, out), decoded(codes, scales).to(out))
    (c, s), (ct, st), parts = fp8.tile_codes(x, True, True, True)
    assert torch.equal(c.view(torch.uint8), raw) and torch.equal(decoded(c, s).cpu(), ref)
    assert torch.equal(decoded(ct, st).cpu(), definition(x, 128, 1)[0].t())
    stored = ct.view(torch.uint8).as_strided((cols, ct.stride(0)), (ct.stride(0), 1))
    assert not stored[:, rows:].any()
    sums = x.double().sum(0)
    assert bool(((fp8.join_sums(parts, torch.float32).double() - sums).abs() <= (rows + 1) * 2.0 ** -24 * x.double().abs().sum(0)).all())
    c, s, ct, st = fp8.quantize_weight(x, both=True)
    square = definition(x, 128, 128)[0]
    assert torch.equal(decoded(c, s).cpu(), square) and torch.equal(decoded(ct, st).cpu(), square.t())
    only = fp8.quantize_weight(x)
    assert torch.equal(only[0].view(torch.uint8), c.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite_stay_apart(cuda_device, dtype, bad):
    from actnn_b200.cpp_extension import fp8
    x = tokens(200, 300, dtype)
    for at in ((2, 77), (2, 78), (130, 299), (131, 0)):
        x[at] = bad
    assert same(decoded(*fp8.quantize(x)).cpu(), definition(x, 1, 128)[0])
    _, there, _ = fp8.tile_codes(x)
    assert same(decoded(*there).cpu(), definition(x, 128, 1)[0].t())
    w = fp8.quantize_weight(x, both=True)
    assert same(decoded(*w[:2]).cpu(), definition(x, 128, 128)[0]) and same(decoded(*w[2:]).cpu(), definition(x, 128, 128)[0].t())
    clean = tokens(200, 300, dtype)
    y, want = (fp8.linear(clean[:5], *w[:2]), fp8.linear(clean[:5], *fp8.quantize_weight(torch.where(x.isfinite(), x, torch.zeros_like(x)))))
    rows = [2, 130, 131]
    keep = [i for i in range(200) if i not in rows]
    assert y[:, rows].isnan().all() and torch.equal(y[:, keep], want[:, keep])
    for t in (5, 200):                                  # one launch, and two
        y = fp8.linear(x[:t], *fp8.quantize_weight(clean))
        assert y[2].isnan().all() and not y[[0, 1, 3, 4]].isnan().any()


def test_tiny_and_huge_blocks(cuda_device):
    from actnn_b200.cpp_extension import fp8
    x = torch.ones(6, 128, device="cuda")
    for i, v in enumerate((1e-42, 3.4e38, 1e-38, 448 * 2.0 ** 30, 449 * 2.0 ** 30, 0.0)):
        x[i] = v
    codes, scales = fp8.quantize(x)
    assert torch.equal(decoded(codes, scales).cpu(), definition(x, 1, 128)[0].float().double())      # 2^128 is infinite in fp32
    # scales whose product is beyond fp32 although the result is not
    w = torch.full((16, 128), 2.0 ** 120, device="cuda")
    y = fp8.linear(torch.full((1, 128), 2.0 ** -120, device="cuda"), *fp8.quantize_weight(w))
    assert torch.equal(y, torch.full_like(y, 128.0))
    y = fp8.linear(torch.zeros(1, 128, device="cuda"), *fp8.quantize_weight(w))
    assert torch.equal(y, torch.zeros_like(y))


@pytest.mark.parametrize("dtype", DTYPES)
def test_matrices_of_other_strides(cuda_device, dtype):
    from actnn_b200.cpp_extension import fp8
    base = tokens(40, 96, dtype)
    for x in (base[:, 8:72], base[:, 3:50], base[::2], base[1:, 1:], base.t(), base[:1].expand(7, 96), base[:, :1]):
        ref = definition(x.contiguous(), 1, 128)[0]
        assert torch.equal(decoded(*fp8.quantize(x)).cpu(), ref)
        here, there, _ = fp8.tile_codes(x)
        assert torch.equal(decoded(*here).cpu(), ref) and torch.equal(decoded(*there).cpu(), definition(x.contiguous(), 128, 1)[0].t())
    for x in (base.view(4, 10, 96), base.view(4, 10, 96).transpose(0, 1)):
        codes, scales = fp8.quantize(x)
        assert codes.shape == x.shape and torch.equal(decoded(codes, scales).cpu().view(40, 96), definition(x.reshape(40, 96), 1, 128)[0])


# sizes of every cut: single tokens, one tile, several, shared reductions of two to eight, pairs, wide accumulators, odd widths
PRODUCTS = [(1, 1, 1), (1, 128, 128), (1, 1000, 2048), (2, 33, 500), (3, 260, 129), (8, 4096, 96), (8, 100, 9000), (9, 300, 1001), (16, 128, 127),
            (17, 129, 1025), (31, 500, 640), (33, 130, 5000), (64, 70, 4096), (100, 1000, 777), (100, 2048, 8192), (129, 640, 130), (192, 256, 384),
            (193, 256, 384), (224, 1024, 512), (225, 257, 385), (256, 1024, 1024), (257, 127, 2000), (300, 1024, 8192), (400, 8192, 640), (448, 512, 128),
            (600, 1111, 300), (1000, 4096, 1024), (1025, 2000, 144), (2048, 4096, 512), (3000, 1500, 264), (5000, 1000, 264), (6000, 4100, 300)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,n,k", PRODUCTS)
def test_product(cuda_device, dtype, t, n, k):
    from actnn_b200.cpp_extension import fp8
    x, w, b = tokens(t, k, dtype), tokens(n, k, dtype, 1), tokens(1, n, dtype, 2)[0]
    wc, ws = fp8.quantize_weight(w)
    c, s = fp8.quantize(x)
    dx, dw = decoded(c, s), decoded(wc, ws)
    first = fp8.matmul(c, s, wc, ws, b, dtype)
    check_product(first, dx, dw, b)
    check_product(fp8.linear(x, wc, ws, b), dx, dw, b)
    check_product(fp8.linear(x, wc, ws), dx, dw)
    assert torch.equal(fp8.matmul(c, s, wc, ws, b, dtype), first)              # reproducible
    for out in DTYPES:
        check_product(fp8.matmul(c, s, wc, ws, None, out), dx, dw)


def test_operands_and_outputs_of_other_strides(cuda_device):
    from actnn_b200.cpp_extension import fp8
    x, w = tokens(300, 200, torch.bfloat16), tokens(128, 200, torch.bfloat16, 1)
    c, s = fp8.quantize(x)
    wc, ws = fp8.quantize_weight(w)
    want = fp8.matmul(c, s, wc, ws)
    for codes in (c.contiguous(), c.view(torch.uint8).t().contiguous().t().view(CODES)):
        assert torch.equal(fp8.matmul(codes, s, wc, ws), want)
    shifted = torch.empty(s.numel() + 8, dtype=torch.uint8, device="cuda")[8:].view(s.shape).copy_(s)
    assert torch.equal(fp8.matmul(c, shifted, wc, ws), want)
    assert torch.equal(fp8.linear(x.view(3, 100, 200), wc, ws), fp8.linear(x, wc, ws).view(3, 100, 128))
    assert torch.equal(fp8.linear(x[:4], wc.contiguous(), ws), fp8.linear(x[:4], wc, ws))


def test_sums_hold_over_a_long_reduction(cuda_device):
    """All terms of one sign: what is lost at each addition would add up."""
    from actnn_b200.cpp_extension import fp8
    x, w = tokens(40, 65536, torch.bfloat16).abs(), tokens(130, 65536, torch.bfloat16, 1).abs()
    c, s = fp8.quantize(x)
    wc, ws = fp8.quantize_weight(w)
    ref = decoded(c, s) @ decoded(wc, ws).t()
    for y in (fp8.matmul(c, s, wc, ws, None, torch.float32), fp8.linear(x[:1].float(), wc, ws)):
        # 32 terms join the sum at a time: 2048 additions that lose 2^-23 each, and as much again among the 32
        assert float(((y.double() - ref[:y.shape[0]]) / ref[:y.shape[0]]).abs().max()) <= 2.0 ** -11


def coded(x, high, wide):
    return definition(x, high, wide)[0].to(x.device)


@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,n,k", [(1, 40, 64), (7, 130, 100), (33, 64, 256), (200, 300, 129), (513, 640, 384), (1200, 513, 1000)])
def test_gradients(cuda_device, dtype, t, n, k, with_bias):
    from actnn_b200 import ops
    x, w, b, dy = (v.requires_grad_() for v in (tokens(t, k, dtype), tokens(n, k, dtype, 1), tokens(1, n, dtype, 2)[0], tokens(t, n, dtype, 3)))
    dy = dy.detach()
    y = ops.fp8_linear.apply(x, w, b if with_bias else None)
    grads = torch.autograd.grad(y, (x, w) + ((b,) if with_bias else ()), dy)
    wq = coded(w, 128, 128)
    check_product(y.detach(), coded(x, 1, 128), wq, b.detach() if with_bias else None)
    check_product(grads[0], coded(dy, 1, 128), wq.t())
    check_product(grads[1], coded(dy, 128, 1).t(), coded(x, 128, 1).t())
    if with_bias:
        sums = dy.double().sum(0)
        assert bool(((grads[2].double() - sums).abs() <= UNIT[dtype] * sums.abs() + (t + 1) * 2.0 ** -23 * dy.double().abs().sum(0)).all())
    # against differences of the layer itself, which is linear in each argument: every operand of a product is off by at most 2^-4 of itself,
    # or 2^-10 of 2^e, where its block's largest magnitude is above 224 * 2^e
    dx, dw = dy.double() @ w.double(), dy.double().t() @ x.double()

    def room(a, high, wide):
        rows, cols = a.shape
        full = torch.nn.functional.pad(a.double().abs(), (0, -cols % wide, 0, -rows % high)).view((rows + high - 1) // high, high, -1, wide)
        step = full.amax((1, 3), keepdim=True) * (2.0 ** -10 / 224)
        return torch.maximum(full * 2.0 ** -4, step).view((rows + high - 1) // high * high, -1)[:rows, :cols]

    def slack(a, b, da, db):
        return (da @ b.abs() + a.abs() @ db + da @ db)

    for got, want, bound in ((grads[0], dx, slack(dy.double(), w.double(), room(dy, 1, 128), room(w, 128, 128))),
                             (grads[1], dw, slack(dy.double().t(), x.double(), room(dy, 128, 1).t(), room(x, 128, 1)))):
        assert bool(((got.double() - want).abs() <= bound * (1 + 2.0 ** -6) + UNIT[dtype] * want.abs() + 2.0 ** -24).all())


@pytest.mark.parametrize("half", ["native", "python"])
@pytest.mark.parametrize("flags", [(True, True, True), (True, False, False), (False, True, False), (False, False, True), (True, False, True)])
def test_only_what_a_gradient_needs_is_kept(cuda_device, monkeypatch, flags, half):
    from actnn_b200 import _lib, ops
    from test_swap_token_inputs_gpu import held
    if half == "python":
        monkeypatch.setattr(_lib, "_native", False)
    t, k, n = 4096, 1024, 512
    x, w, b = tokens(t, k, torch.float16), tokens(n, k, torch.float16, 1), tokens(1, n, torch.float16, 2)[0]
    dy = tokens(t, n, torch.float16, 3)
    every = [v.clone().requires_grad_() for v in (x, w, b)]
    ops.fp8_linear.apply(*every).backward(dy)
    mine = [v.requires_grad_(f) for v, f in zip((x, w, b), flags)]
    before = held()
    y = ops.fp8_linear.apply(*mine)
    kept = held() - before - y.numel() * 2
    needed = flags[0] * (n * k + n * k // 128) + flags[1] * (t * k + t * k // 128)
    assert needed <= kept <= needed + 4096
    y.backward(dy)
    for got, want, asked in zip(mine, every, flags):
        assert torch.equal(got.grad, want.grad) if asked else got.grad is None


@pytest.mark.parametrize("half", ["native", "python"])
@pytest.mark.parametrize("t,k,n", [(0, 32, 8), (5, 0, 8), (5, 32, 0), (0, 0, 0)])
def test_empty_dimensions(cuda_device, monkeypatch, t, k, n, half):
    from actnn_b200 import _lib, ops
    if half == "python":
        monkeypatch.setattr(_lib, "_native", False)
    x, w, b = (torch.randn(*s, device="cuda").half().requires_grad_() for s in ((t, k), (n, k), (n,)))
    y = ops.fp8_linear.apply(x, w, b)
    assert y.shape == (t, n) and torch.equal(y, b.detach().expand(t, n))
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert gx.shape == x.shape and gw.shape == w.shape and torch.equal(gb, torch.full_like(gb, t))
    assert not gx.any() and not gw.any()


def test_a_gradient_that_is_expanded_or_transposed(cuda_device):
    from actnn_b200 import ops
    x, w = tokens(130, 96, torch.bfloat16), tokens(72, 96, torch.bfloat16, 1)
    leaves = [v.clone().requires_grad_() for v in (x, w)]
    y = ops.fp8_linear.apply(*leaves)
    for dy in (torch.ones((), device="cuda", dtype=torch.bfloat16).expand(130, 72), tokens(72, 130, torch.bfloat16, 3).t()):
        got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        want = torch.autograd.grad(y, leaves, dy.contiguous(), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("t", [1, 10, 200])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_layer(cuda_device, dtype, t, with_bias):
    """Frozen and not, with autocast and without: the type and the values (the sums of few tokens go in another order)."""
    import actnn_b200 as actnn
    layer = actnn.QFp8Linear(96, 72, with_bias).cuda().eval()
    x = tokens(t, 96, torch.float32)
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
        want = layer(x)
        got = layer.freeze()(x)
    assert got.dtype == want.dtype == dtype
    check_product(got, coded(x.to(dtype), 1, 128), coded(layer.weight.detach().to(dtype), 128, 128), layer.bias.detach().to(dtype) if with_bias else None)
    if t > 8:
        assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="frozen"):
        layer(x.requires_grad_())
    layer.train()
    assert layer.frozen is None
    layer(x).sum().backward()
    assert layer.weight.grad.shape == layer.weight.shape and x.grad.shape == x.shape
    assert layer.freeze().frozen is not None and layer.half().frozen is None


def test_refusals(cuda_device):
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import fp8
    x, w = tokens(4, 32, torch.float16), tokens(8, 32, torch.float16, 1)
    c, s = fp8.quantize_weight(w)
    for call, word in ((lambda: fp8.linear(x[:, :16], c, s), "multiplied"), (lambda: fp8.linear(x, c.view(torch.uint8), s), "type"),
                       (lambda: fp8.linear(x, c, s[:, :, :256]), "dimension"), (lambda: fp8.linear(x, c, s, x[0]), "dimension of bias"),
                       (lambda: fp8.linear(x, c, s.int()), "type"), (lambda: fp8.linear(x.double(), c, s), "type of x"),
                       (lambda: ops.fp8_linear.apply(x, w[:, :16]), "multiplied"), (lambda: ops.fp8_linear.apply(x, w, x[0]), "dimension of bias"),
                       (lambda: fp8.matmul(c, s, c[:, :16], s), "multiplied"), (lambda: fp8.quantize_weight(x[0]), "dimension"),
                       (lambda: fp8.linear(x, c, s, w[:, 0].cpu()), "CUDA")):
        with pytest.raises(RuntimeError, match=word):
            call()


def captured(run):
    """A graph of `run` and what it returned."""
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    return graph, out


def test_captured_and_replayed(cuda_device):
    """Two graphs of the same calls, replayed one after the other on changed inputs, beside calls that are not captured."""
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import fp8
    x, w, b, dy = tokens(300, 256, torch.bfloat16), tokens(192, 256, torch.bfloat16, 1), tokens(1, 192, torch.bfloat16, 2)[0], tokens(300, 192, torch.bfloat16, 3)
    code = fp8.quantize_weight(w)

    def run():
        leaves = [v.detach().requires_grad_() for v in (x, w, b)]
        y = ops.fp8_linear.apply(*leaves)
        return (y.detach(), fp8.linear(x, *code, b), fp8.linear(x[:3], *code, b)) + torch.autograd.grad(y, leaves, dy)

    one, two_ = captured(run), captured(run)
    for seed in (5, 6):
        x.copy_(tokens(300, 256, torch.bfloat16, seed))
        dy.copy_(tokens(300, 192, torch.bfloat16, seed + 10))
        want = run()
        for graph, out in (one, two_):
            graph.replay()
            assert all(torch.equal(a, v) for a, v in zip(out, want))


def test_calls_on_two_streams_at_once(cuda_device):
    from actnn_b200.cpp_extension import fp8
    x, w = tokens(500, 1024, torch.bfloat16), tokens(2048, 1024, torch.bfloat16, 1)
    code = fp8.quantize_weight(w)
    want = fp8.linear(x, *code), fp8.linear(x[:200], *code)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(fp8.linear(x if i == 0 else x[:200], *code))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,n,k", [(1, 40, 64), (7, 130, 100), (33, 64, 256), (300, 200, 384)])
def test_both_halves_of_the_binding_agree(cuda_device, monkeypatch, dtype, t, n, k):
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import fp8
    from test_token_bindings_gpu import both_halves, grads
    x, w, b = tokens(t, k, dtype), tokens(n, k, dtype, 1), tokens(1, n, dtype, 2)[0]
    code = fp8.quantize_weight(w)
    both_halves(monkeypatch, lambda: [fp8.linear(x, *code, b), fp8.linear(x.view(1, t, k), *code)])
    both_halves(monkeypatch, lambda: grads(ops.fp8_linear.apply, (x, w, b)))


def test_swapped_codes_give_the_same_gradients(cuda_device):
    import actnn_b200 as actnn
    from actnn_b200 import ops
    from test_token_bindings_gpu import grads
    x, w, b = tokens(257, 384, torch.bfloat16), tokens(192, 384, torch.bfloat16, 1), tokens(1, 192, torch.bfloat16, 2)[0]
    want = grads(ops.fp8_linear.apply, (x, w, b))
    actnn.set_optimization_level("L4")
    assert all(torch.equal(a, v) for a, v in zip(grads(ops.fp8_linear.apply, (x, w, b)), want))


def test_sums_of_columns_that_are_not_finite(cuda_device):
    from actnn_b200.cpp_extension import fp8
    x = tokens(300, 200, torch.bfloat16)
    x[5, 3], x[130, 4], x[131, 4], x[7, 5] = float("inf"), float("inf"), -float("inf"), float("nan")
    sums = fp8.join_sums(fp8.tile_codes(x, True, True, True)[2], torch.float32).double().cpu()
    want = x.double().sum(0).cpu()
    assert sums[3] == float("inf") and sums[4].isnan() and sums[5].isnan()
    keep = want.isfinite()
    assert int(keep.sum()) == 197 and bool(((sums - want)[keep].abs() <= 301 * 2.0 ** -24 * x.double().abs().sum(0).cpu()[keep]).all())
