"""The two halves of the binding give the same results for the token operators, to the bit: the C++ functions, and the Python
ones that run where another build of the library is asked for."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def both_halves(monkeypatch, run):
    from actnn_b200 import _lib
    first = run()
    with monkeypatch.context() as m:
        m.setattr(_lib, "_native", False)
        second = run()
    assert len(first) == len(second)
    for a, b in zip(first, second):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


def grads(call, leaves, dy_like=None):
    leaves = [v.detach().clone().requires_grad_() for v in leaves]
    y = call(*leaves)
    g = torch.Generator(device="cuda").manual_seed(5)
    y.backward(torch.randn(y.shape, generator=g, device="cuda").to(y.dtype))
    return [y.detach()] + [v.grad for v in leaves]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,n,k", [(1, 40, 64), (7, 130, 100), (33, 64, 256)])
def test_int8_linear(cuda_device, monkeypatch, dtype, t, n, k):
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import int8
    torch.manual_seed(0)
    x, w, b = (torch.randn(*s, device="cuda").to(dtype) for s in ((t, k), (n, k), (n,)))
    code = int8.quantize_rows(w)
    both_halves(monkeypatch, lambda: [int8.linear(x, *code, b), int8.linear(x.view(1, t, k), *code)])
    both_halves(monkeypatch, lambda: grads(ops.int8_linear.apply, (x, w, b)))


@pytest.mark.parametrize("level", ["L3", "L0"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_activations(cuda_device, monkeypatch, dtype, level):
    import actnn_b200 as actnn
    from actnn_b200 import ops
    actnn.set_optimization_level(level)
    x = torch.randn(9, 130, device="cuda").to(dtype)
    for name in ("relu", "silu", "gelu", "gelu_tanh"):
        both_halves(monkeypatch, lambda: grads(lambda v: ops.activation.apply(v, name), (x,)))
        both_halves(monkeypatch, lambda: grads(lambda v: ops.glu.apply(v, name), (x,)))


@pytest.mark.parametrize("level", ["L3", "L0"])
@pytest.mark.parametrize("shape,groups", [((2, 32, 9, 9), 4), ((3, 30, 5), 3), ((300, 64, 14, 14), 8)])
def test_group_norm(cuda_device, monkeypatch, shape, groups, level):
    import actnn_b200 as actnn
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import group_norm
    actnn.set_optimization_level(level)
    x, w, b = torch.randn(shape, device="cuda").half(), torch.randn(shape[1], device="cuda"), torch.randn(shape[1], device="cuda")
    both_halves(monkeypatch, lambda: [group_norm.inference(x, groups, w, b, 1e-5, "gelu")])
    both_halves(monkeypatch, lambda: grads(lambda v, p, q: ops.group_norm.apply(v, groups, p, q, 1e-5, "silu"), (x, w, b)))
    both_halves(monkeypatch, lambda: grads(lambda v: ops.group_norm.apply(v, groups, None, None, 1e-5, None), (x,)))
