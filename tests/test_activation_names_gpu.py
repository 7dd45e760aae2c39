"""No activation, as None or as "none": the same everywhere."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("half", ["native", "python"])
def test_none(cuda_device, monkeypatch, half):
    import actnn_b200 as actnn
    from actnn_b200 import _lib, ops
    if half == "python":
        monkeypatch.setattr(_lib, "_native", False)
    x = torch.randn(6, 32, device="cuda", requires_grad=True)
    for call in (ops.activation.apply, ops.glu.apply, lambda v, name: ops.group_norm.apply(v, 4, name=name),
                 lambda v, name: actnn.QGLU(name)(v), lambda v, name: actnn.QGroupNorm(4, 32, activation=name).cuda()(v)):
        got, want = call(x, None), call(x, "none")
        assert torch.equal(got, want)
        (g,), (w,) = torch.autograd.grad(got.sum(), x), torch.autograd.grad(want.sum(), x)
        assert torch.equal(g, w)
    assert repr(actnn.QGLU(None)) == repr(actnn.QGLU("none"))
    for bad in (3, "swish", ["silu"]):
        for call in (ops.activation.apply, ops.glu.apply, lambda v, name: ops.group_norm.apply(v, 4, name=name)):
            with pytest.raises(RuntimeError, match="activation must be one of"):
                call(x, bad)
