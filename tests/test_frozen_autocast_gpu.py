"""A frozen QInt8Linear under autocast gives what the layer that is not frozen gives: the type, and the values."""
import pytest
import torch

from test_int8_linear_gpu import tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("t", [1, 10, 200])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_same_output(cuda_device, dtype, t, with_bias):
    import actnn_b200 as actnn
    layer = actnn.QInt8Linear(96, 72, with_bias).cuda().eval()
    x = tokens(t, 96, torch.float32)
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
        want = layer(x)
        got = layer.freeze()(x)
    assert got.dtype == want.dtype == dtype and torch.equal(got, want)
    with torch.no_grad():
        layer.unfreeze()
        want = layer(x)
        assert want.dtype == torch.float32 and torch.equal(layer.freeze()(x), want)
        with torch.autocast("cuda", dtype=dtype):        # codes of the weight as it was where freeze() was called
            assert layer(x).dtype == dtype
