"""The 8-bit floating-point layer where no gradients are recorded: leaves ask for theirs all the same, and nothing is coded for them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("half", ["native", "python"])
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
@pytest.mark.parametrize("t", [5, 2048])
def test_nothing_is_made_for_gradients_that_cannot_come(cuda_device, monkeypatch, t, mode, half):
    import actnn_b200 as actnn
    from actnn_b200 import _lib
    from test_fp8_linear_gpu import tokens
    if half == "python":
        monkeypatch.setattr(_lib, "_native", False)
    k, n = 1024, 512
    layer = actnn.QFp8Linear(k, n).cuda().half()
    layer.eval()                                             # not frozen: an evaluation between two epochs
    x = tokens(t, k, torch.float16).requires_grad_()
    want = layer(x)

    def stat(which):
        return torch.cuda.memory_stats()["requested_bytes.all." + which]

    with mode():
        got = layer(x)
        assert not got.requires_grad and torch.equal(got, want)
        got = None
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = stat("current")
        layer(x)
        most = stat("peak") - before
    scales = (t + 127) // 128 * 128 * (k // 128) + n * (k // 128)
    needed = 2 * t * n + t * k + n * k + scales              # the result and one set of codes of each operand
    assert needed <= most <= needed + 4096
    # where gradients are recorded they are what they were
    want.sum().backward()
    assert x.grad.shape == x.shape and layer.weight.grad.shape == layer.weight.shape and layer.bias.grad.shape == (n,)
