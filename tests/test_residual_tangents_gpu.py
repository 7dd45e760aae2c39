"""Forward-mode derivatives of the operators of a residual branch: none is passed on, and none is dropped in silence."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

NAMES = "x branch weight bias post_weight post_bias gate".split()


@pytest.mark.parametrize("half", ["native", "python"])
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", NAMES)
def test_norms(cuda_device, monkeypatch, which, grad, half):
    from actnn_b200 import _lib, ops
    from actnn_b200.cpp_extension import residual_norm
    if half == "python":
        monkeypatch.setattr(_lib, "_native", False)
    values = [torch.randn(4, 16, device="cuda") for _ in range(2)] + [torch.randn(16, device="cuda") for _ in range(5)]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        want = ops.residual_norm.apply(*values, kind="layer")              # nothing has a tangent
        i = NAMES.index(which)
        dual = values[:i] + [forward_ad.make_dual(values[i], torch.ones_like(values[i]))] + values[i + 1:]
        for call in (lambda: ops.residual_norm.apply(*dual, kind="layer"), lambda: residual_norm.inference(*dual, kind="layer")):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        for leaf in values:                                                # where gradients are recorded: by autograd's own refusal
            leaf.requires_grad_()
        with pytest.raises((RuntimeError, NotImplementedError)):
            ops.residual_norm.apply(*dual, kind="layer")
        for leaf in values:
            leaf.requires_grad_(False)
        got = ops.residual_norm.apply(*values, kind="layer")
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("half", ["native", "python"])
def test_product_and_dropout(cuda_device, monkeypatch, half):
    from actnn_b200 import _lib, ops
    if half == "python":
        monkeypatch.setattr(_lib, "_native", False)
    x, w = torch.randn(4, 32, device="cuda"), torch.randn(8, 32, device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.fp8_linear.apply(dual, w), lambda: ops.seeded_dropout.apply(dual, 0.5)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
