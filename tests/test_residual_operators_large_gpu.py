"""Operators of a residual branch on more than 2^31 elements, against the same call on the last rows alone; and inputs of one, three and four
dimensions against those of two."""
import pytest
import torch

pytestmark = pytest.mark.gpu

MANY = 1 << 31


def filled(rows, cols, dtype=torch.bfloat16):
    """Rows that differ, made in place of random ones: quick, and no temporary of another type."""
    x = torch.empty(rows, cols, dtype=dtype, device="cuda")
    for i in range(0, rows, 8192):
        x[i:i + 8192].normal_(generator=None)
    return x


def test_dropout(cuda_device):
    """The fields of the last elements, from the definition of their calls."""
    from actnn_b200 import ops
    from test_seeded_dropout_gpu import fields
    n, tail, key = MANY + 1003, 4096 + 3, (77, 2 ** 33 + 4)
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda").requires_grad_()
    y = ops.seeded_dropout.apply(x, 0.5, key)
    g, = torch.autograd.grad(y, x, torch.ones_like(x))
    first = (n - tail) // 8 * 8
    calls = torch.arange(first // 8, (n + 7) // 8)
    low, seed, offset = 0xFFFFFFFF, *key
    c = [calls & low, calls >> 32, torch.full_like(calls, offset & low), torch.full_like(calls, offset >> 32)]
    k0, k1 = seed, 0
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [((p1 >> 32) & low) ^ c[1] ^ k0, p1 & low, ((p0 >> 32) & low) ^ c[3] ^ k1, p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    field = torch.stack([(v >> s) & 0xFFFF for v in c for s in (0, 16)], -1).reshape(-1)[:n - first]
    want = torch.where(field >= 32768, 2.0, 0.0).to(torch.bfloat16)
    assert torch.equal(y.detach()[first:].cpu(), want) and torch.equal(g[first:].cpu(), want)
    head = torch.where(fields(4096, key) >= 32768, 2.0, 0.0).to(torch.bfloat16)
    assert torch.equal(y.detach()[:4096].cpu(), head)


@pytest.mark.parametrize("kind,c,p", [("rms", 32768, 0.0), ("layer", 4096, 0.0), ("rms", 1001, 0.1)])
def test_norms(cuda_device, kind, c, p):
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import seeded_dropout
    rows, last = MANY // c + 50, 40
    x, f = filled(rows, c), filled(rows, c)
    w, pw = torch.randn(c, device="cuda").to(torch.bfloat16), torch.randn(c, device="cuda").to(torch.bfloat16)
    key = (5, 12)

    def run(x, f, p):
        leaves = [v.detach().requires_grad_() for v in (x, f)]
        r, h = ops.residual_norm.apply(*leaves, w, None, pw, p=p, kind=kind, key=key)
        gx, gf = torch.autograd.grad((r, h), leaves, (x, f))                   # any gradients of the right shape
        return [v[-last:].clone() for v in (r.detach(), h.detach(), gx, gf)]

    got = run(x, f, p)
    if p == 0:
        want = run(x[-last:].clone(), f[-last:].clone(), p)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    else:                                                    # the mask is that of the element's place in the whole
        keep = seeded_dropout.apply_mask(torch.ones(rows * c, dtype=torch.bfloat16, device="cuda"), p, key).view(rows, c)[-last:] != 0
        f, x = f[-last:].float(), x[-last:].float()
        n = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-5) * pw.float()
        want = x + torch.where(keep, n / (1 - p), torch.zeros_like(n))
        # the rounding to bfloat16; a row's sums, 1001 terms in any order, are off by 2^-14 of themselves at most, a dozen products by 2^-24 each
        assert bool(((got[0].float() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -13 * (n.abs() + x.abs())).all())


def test_codes_and_product(cuda_device):
    from actnn_b200.cpp_extension import fp8
    cols = 8192
    rows = MANY // cols + 131
    x = filled(rows, cols)
    last = 131
    codes, scales = fp8.quantize(x)
    c, s = fp8.quantize(x[-last:].clone())
    assert torch.equal(codes.view(torch.uint8)[-last:], c.view(torch.uint8))
    assert torch.equal(fp8.dequantize(codes, scales)[-last:], fp8.dequantize(c, s))
    (rc, _), (tc, ts), _ = fp8.tile_codes(x)
    assert torch.equal(rc.view(torch.uint8), codes.view(torch.uint8))
    first = rows // 128 * 128                                # a block of tokens of its own
    (_, _), (tail, tail_s), _ = fp8.tile_codes(x[first:].clone())
    assert torch.equal(tc.view(torch.uint8)[:, first:], tail.view(torch.uint8))
    rc = tc = tail = None
    w, ws = fp8.quantize_weight(torch.randn(72, cols, device="cuda").to(torch.bfloat16))
    y, part = fp8.matmul(codes, scales, w, ws, None, torch.float32), fp8.matmul(c, s, w, ws, None, torch.float32)
    # cut in another way, sums in another order: each is off by 2^-23 of the magnitudes for each addition, rounded or cut off
    mag = fp8.dequantize(c, s, torch.float32).double().abs() @ fp8.dequantize(w, ws, torch.float32).double().abs().t()
    assert bool(((y[-last:].double() - part.double()).abs() <= 2 * (cols + 2) * 2.0 ** -23 * mag).all())


def test_results_past_32_bits(cuda_device):
    from actnn_b200.cpp_extension import fp8
    k, n = 64, 16384
    t = MANY // n + 300
    x = filled(t, k)
    w, ws = fp8.quantize_weight(torch.randn(n, k, device="cuda").to(torch.bfloat16))
    y = fp8.linear(x, w, ws)
    part = fp8.linear(x[-300:].clone(), w, ws)
    assert torch.equal(y[-300:], part)                       # one block of the reduction: one order of its sums


@pytest.mark.parametrize("half", ["native", "python"])
@pytest.mark.parametrize("lead", [(), (5,), (3, 7), (2, 3, 5)])
def test_inputs_of_any_dimensions(cuda_device, monkeypatch, lead, half):
    from actnn_b200 import _lib, ops
    from actnn_b200.cpp_extension import fp8, residual_norm
    if half == "python":
        monkeypatch.setattr(_lib, "_native", False)
    k, n = 96, 40
    rows = torch.Size(lead).numel()
    x, f, dy = torch.randn(rows, k, device="cuda"), torch.randn(rows, k, device="cuda"), torch.randn(rows, n, device="cuda")
    w, b, g = torch.randn(n, k, device="cuda"), torch.randn(n, device="cuda"), torch.randn(k, device="cuda")

    def both(call, inputs, outs):
        """The call on two dimensions and on all, its gradients too."""
        results = []
        for shape in ((rows,), lead):
            leaves = [v.view(shape + v.shape[1:]).detach().requires_grad_() for v in inputs]
            y = call(*leaves)
            y = y if isinstance(y, tuple) else (y,)
            assert all(v.shape == tuple(shape) + v.shape[-1:] for v in y)
            grads = torch.autograd.grad(y, leaves, [d.view(shape + d.shape[1:]) for d in outs])
            results.append([v.detach().reshape(rows, -1) for v in y + grads])
        assert all(torch.equal(a, v) for a, v in zip(*results))

    both(lambda v: ops.fp8_linear.apply(v, w, b), [x], [dy])
    both(lambda v: ops.seeded_dropout.apply(v, 0.3, (1, 4)), [x], [x])
    both(lambda v, u: ops.residual_norm.apply(v, u, g, None, g, None, g, p=0.2, key=(3, 4)), [x, f], [f, x])
    code = fp8.quantize_weight(w)
    assert torch.equal(fp8.linear(x.view(lead + (k,)), *code, b).reshape(rows, n), fp8.linear(x, *code, b))
    c, s = fp8.quantize(x.view(lead + (k,)))
    assert c.shape == lead + (k,) and torch.equal(fp8.dequantize(c, s).reshape(rows, k), fp8.dequantize(*fp8.quantize(x)))
    assert torch.equal(fp8.matmul(c, s, *code, b).reshape(rows, n), fp8.matmul(*fp8.quantize(x), *code, b))
    for a, v in zip(residual_norm.inference(x.view(lead + (k,)), f.view(lead + (k,)), g), residual_norm.inference(x, f, g)):
        assert torch.equal(a.reshape(rows, k), v)
