"""The operators of a residual branch together, as examples/residual_block.py uses them."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT
from test_fp8_linear_gpu import captured, definition

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("residual_block", os.path.join(ROOT, "examples", "residual_block.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


class Product(torch.autograd.Function):
    """The product of codes in 64 bits, with the gradients of the codes."""

    @staticmethod
    def coded(v, high, wide):
        return definition(v.float(), high, wide)[0].to(v.device)

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return Product.coded(x, 1, 128) @ Product.coded(w, 128, 128).t()

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        return Product.coded(dy, 1, 128) @ Product.coded(w, 128, 128), Product.coded(dy, 128, 1).t() @ Product.coded(x, 128, 1)


def plain(model, x, layer):
    """The stack without dropout in 64 bits."""
    def norm(v, w, b):
        m = v.mean(-1, keepdim=True) if layer else 0.0
        y = (v - m) / torch.sqrt(((v - m) ** 2).mean(-1, keepdim=True) + 1e-5) * w
        return y + b if layer else y

    p = {n: v.detach().double().requires_grad_() for n, v in model.named_parameters()}
    r = h = x
    for i in range(len(model.blocks)):
        q = {n.split(".", 2)[2]: v for n, v in p.items() if n.startswith("blocks.%d." % i)}
        a, b = (Product.apply(h, q["up.weight"]) + q["up.bias"]).chunk(2, -1)
        f = Product.apply(torch.nn.functional.silu(a) * b, q["down.weight"]) + q["down.bias"]
        r = r + q["norm.gate"] * norm(f, q["norm.post_weight"], q.get("norm.post_bias"))
        h = norm(r, q["norm.weight"], q.get("norm.bias"))
    return h, p


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_gradients(cuda_device, example, kind):
    """In float32 the two differ by 2^-20 or so between products; of the values to be coded a few in 10^5 then round to the neighbouring code,
    an eighth away: 2^-11 of the norm a product, and far fewer than 16 of them on the way to any gradient."""
    import actnn_b200 as actnn
    actnn.set_optimization_level("L0")
    torch.manual_seed(0)
    model = example.Stack(channels=96, hidden=200, kind=kind, p=0.0).cuda().train()
    x, dy = torch.randn(150, 96, device="cuda"), torch.randn(150, 96, device="cuda")
    leaf, wide = x.clone().requires_grad_(), x.double().requires_grad_()
    y = model(leaf)
    y.backward(dy)
    want, p = plain(model, wide, kind == "layer")
    want.backward(dy.double())
    pairs = [("y", y.detach(), want.detach()), ("x", leaf.grad, wide.grad)] + [(n, v.grad, p[n].grad) for n, v in model.named_parameters()]
    for name, got, ref in pairs:
        assert float((got.double() - ref).norm()) <= 2.0 ** -7 * float(ref.norm()), name


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("level", ["L0", "L3", "L4"])
def test_training_runs(cuda_device, example, level, kind):
    losses, kept, model = example.train(3, level, kind)
    assert all(v == v and v < 1e3 for v in losses) and all(bool(p.grad.isfinite().all()) for p in model.parameters())
    import actnn_b200 as actnn
    actnn.config.__dict__.update(actnn.conf.QuantizationConfig().__dict__)
    assert example.train(3, level, kind)[0] == losses                                   # the same steps twice


def test_what_is_kept(cuda_device, example):
    _, kept, _ = example.train(0, "L3")
    t, c, h = 8 * 500, 256, 640
    codes = t * (c + 2 * h + h + 2 * c)                       # of up's input, of the unit's, of down's, of the norm's two
    weights = 3 * c * h
    r = t * c * 2                                             # the residual stream: the next block takes it, and the last one's result
    assert 2 * (codes + weights) <= kept <= 2.1 * (codes + weights) + 2 * r


def test_swapped_activations_give_the_same_steps(cuda_device, example):
    import actnn_b200 as actnn
    here = example.train(4, "L3")[0]
    actnn.config.__dict__.update(actnn.conf.QuantizationConfig().__dict__)
    assert example.train(4, "L4")[0] == here


@pytest.mark.parametrize("p", [0.0, 0.2])
def test_a_captured_step(cuda_device, example, p):
    model = example.Stack(channels=96, hidden=200, kind="layer", p=p).cuda().bfloat16().train()
    x, dy = (torch.randn(150, 96, device="cuda").bfloat16() for _ in range(2))
    params = list(model.parameters())

    def step():
        leaf = x.detach().requires_grad_()
        y = model(leaf)
        return (y.detach(),) + torch.autograd.grad(y, [leaf] + params, dy)

    graph, out = captured(step)
    seen = []
    for _ in range(2):
        x.copy_(torch.randn(150, 96, device="cuda"))
        graph.replay()
        seen.append([o.clone() for o in out])
        assert all(bool(o.isfinite().all()) for o in out)
        if p == 0:
            assert all(torch.equal(a, b) for a, b in zip(out, step()))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, seen[1])) == (p == 0)             # every replay drops other elements


def test_served_tokens(cuda_device, example):
    model = example.Stack().cuda().bfloat16().eval()
    tokens = torch.randn(33, 256, device="cuda").bfloat16()
    with torch.no_grad():
        want = model(tokens)
        model.freeze()
        assert torch.equal(model(tokens), want)
        for t in (1, 3, 8, 20):
            got = example.Server(model, t, 256)(tokens[:t])
            assert torch.equal(got, model(tokens[:t]))
            # the sums of up to eight tokens go in another order: a bf16 rounding or a code apart here and there
            assert float((got.double() - want[:t].double()).norm()) <= 2.0 ** -6 * float(want[:t].double().norm())


def test_command(cuda_device, example, capsys):
    example.main(["--steps", "2"])
    out = capsys.readouterr().out
    assert "loss" in out and "one token: (1, 256)" in out
