"""Dropout whose mask is never stored: against the dropout that stores it, and against its definition."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def fields(count, key):
    """The 16-bit fields of the generator, in Python integers of 64 bits on the CPU."""
    seed, offset = key
    low = 0xFFFFFFFF
    calls = torch.arange((count + 7) // 8)
    c = [calls & low, calls >> 32, torch.full_like(calls, offset & low), torch.full_like(calls, (offset >> 32) & low)]
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [((p1 >> 32) & low) ^ c[1] ^ k0, p1 & low, ((p0 >> 32) & low) ^ c[3] ^ k1, p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([(v >> s) & 0xFFFF for v in c for s in (0, 16)], -1).reshape(-1)[:count]


def definition(x, p, key):
    """Kept elements times 1 / (1 - p), one rounded fp32 product and one rounding to the type."""
    p32 = float(torch.tensor(p, dtype=torch.float32))
    keep = (fields(x.numel(), key) + 1 > 65536 * p32).view(x.shape)
    inv = torch.tensor(1 / (1 - p32), dtype=torch.float32)
    return torch.where(keep, (x.cpu().float() * inv).to(x.dtype), torch.zeros((), dtype=x.dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 1001), (2, 3, 5, 7), (300, 4096), ()])
@pytest.mark.parametrize("p", [0.0, 1e-6, 0.1, 0.5, 0.99])
def test_values_and_gradients(cuda_device, dtype, shape, p):
    from actnn_b200 import ops
    x, dy = torch.randn(shape, device="cuda").to(dtype).requires_grad_(), torch.randn(shape, device="cuda").to(dtype)
    for key in ((1234, 8), (0xFFFFFFFFFFFFFFFF, 2 ** 40 + 12)):
        y = ops.seeded_dropout.apply(x, p, key)
        gx, = torch.autograd.grad(y, (x,), dy)
        assert torch.equal(y.detach().cpu(), definition(x.detach(), p, key)) and torch.equal(gx.cpu(), definition(dy, p, key))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("numel", [77 * 1001, 5_000_011])
def test_the_same_as_the_dropout_with_a_mask(cuda_device, dtype, numel):
    """From the same state of the generator, which both leave in the same state."""
    import actnn_b200 as actnn
    x = torch.randn(numel, device="cuda").to(dtype)
    torch.manual_seed(11)
    want = actnn.QDropout(0.3).train()(x), torch.rand(4, device="cuda")
    torch.manual_seed(11)
    got = actnn.QSeededDropout(0.3).train()(x), torch.rand(4, device="cuda")
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(actnn.QSeededDropout(0.3).eval()(x), x)


@pytest.mark.parametrize("numel", [2 ** 25 + 5])
def test_large(cuda_device, numel):
    """Several octets a thread; the tail."""
    from actnn_b200.cpp_extension import seeded_dropout
    x = torch.ones(numel, device="cuda", dtype=torch.bfloat16)
    y = seeded_dropout.apply_mask(x, 0.25, (5, 4))
    assert torch.equal(y.cpu(), definition(x, 0.25, (5, 4)))


def test_dropped_elements_are_zero_whatever_they_were(cuda_device):
    from actnn_b200.cpp_extension import seeded_dropout
    for v in (float("nan"), float("inf"), -float("inf")):
        y = seeded_dropout.apply_mask(torch.full((4096,), v, device="cuda"), 0.5, (1, 4))
        kept = (fields(4096, (1, 4)) + 1 > 32768).cuda()
        assert torch.equal(y[~kept], torch.zeros_like(y[~kept])) and not y[kept].isfinite().any()


def test_strides_and_alignment(cuda_device):
    from actnn_b200 import ops
    base = torch.randn(40, 64, device="cuda").half()
    for x in (base.t(), base[:, 1:], base[::2], base.view(-1)[1:], base[:1].expand(5, 64), base.view(4, 4, 10, 16).contiguous(memory_format=torch.channels_last)):
        x = x.detach().requires_grad_()
        y = ops.seeded_dropout.apply(x, 0.4, (3, 8))
        assert torch.equal(y.detach().cpu(), definition(x.detach().contiguous(), 0.4, (3, 8)))
        dy = torch.randn(y.shape[::-1], device="cuda").half().permute(*range(y.dim() - 1, -1, -1))       # a gradient that lies the other way
        assert torch.equal(torch.autograd.grad(y, (x,), dy)[0].cpu(), definition(dy.contiguous(), 0.4, (3, 8)))


def test_nothing_of_an_element_is_kept(cuda_device):
    from actnn_b200 import ops
    from test_swap_token_inputs_gpu import held
    x = torch.randn(1 << 20, device="cuda", requires_grad=True)
    h = x * 1
    before = held()
    y = ops.seeded_dropout.apply(h, 0.5)
    assert held() - before <= y.numel() * 4 + 512
    y.sum().backward()


def test_empty(cuda_device):
    from actnn_b200 import ops
    x = torch.empty(0, 5, device="cuda", requires_grad=True)
    y = ops.seeded_dropout.apply(x, 0.5)
    assert y.shape == (0, 5) and torch.autograd.grad(y, (x,), torch.empty(0, 5, device="cuda"))[0].shape == (0, 5)


def test_replays_of_a_graph_drop_other_elements(cuda_device):
    """Forward and backward of one replay drop the same ones; a seed repeats the sequence; two graphs do not disturb one another."""
    from actnn_b200 import ops
    x, dy = torch.ones(50_000, device="cuda"), torch.ones(50_000, device="cuda")

    def run():
        leaf = x.detach().requires_grad_()
        y = ops.seeded_dropout.apply(leaf, 0.5)
        z = ops.seeded_dropout.apply(leaf, 0.5)
        return (y.detach(), z.detach()) + torch.autograd.grad((y, z), (leaf,), (dy, 10 * dy))

    from test_fp8_linear_gpu import captured
    one, two = captured(run), captured(run)
    seen = []
    for seed in (7, 7):
        torch.manual_seed(seed)
        for graph, (y, z, g) in (one, two, one):
            graph.replay()
            assert torch.equal(g, y + 10 * z) and not torch.equal(y, z) and 0.45 < float((y > 0).float().mean()) < 0.55
            seen.append(y.clone())
    assert all(torch.equal(seen[i], seen[i + 3]) for i in range(3))
    assert not any(torch.equal(seen[i], seen[j]) for i in range(3) for j in range(i))


@pytest.mark.parametrize("dtype", DTYPES)
def test_both_halves_of_the_binding_agree(cuda_device, monkeypatch, dtype):
    from actnn_b200 import ops
    from test_token_bindings_gpu import both_halves, grads
    x = torch.randn(33, 77, device="cuda").to(dtype)
    both_halves(monkeypatch, lambda: grads(lambda v: ops.seeded_dropout.apply(v, 0.3, (9, 4)), (x,)))

    def drawn():
        torch.manual_seed(3)
        return grads(lambda v: ops.seeded_dropout.apply(v, 0.3), (x,))
    both_halves(monkeypatch, drawn)
