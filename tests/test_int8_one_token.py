"""One token through the integer linear layer at every length of the reduction: up to the codes that a launch's shared memory holds
without being asked to hold more, and beyond, where the codes go through a workspace."""
import ctypes

import pytest
import torch

from test_int8_linear_gpu import DTYPES, check_product


def test_codes_and_the_kernels_own_shared_memory_fit_together(built_library):
    """48 KB in all need no opt-in; the kernel has a word for each of up to eight tokens besides the codes."""
    from actnn_b200 import _lib
    lib, size = _lib.load(), ctypes.c_int64(-1)
    for t in range(1, 9):
        for k in list(range(256, 50000, 256)) + [48639, 48640, 48641, 49152, 49153]:
            assert lib.actnn_int8_linear_workspace(t, k, ctypes.addressof(size)) == 0
            if size.value == 0:
                assert t * ((k + 511) // 512 * 512) + 8 * 4 <= 48 * 1024


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [16384, 40000, 48639, 48640, 48641, 49152, 49153, 65536])
def test_product(cuda_device, dtype, k):
    from actnn_b200.cpp_extension import int8
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn(1, k, generator=g, device="cuda").to(dtype)
    weights = torch.randint(-127, 128, (70, (k + 15) // 16 * 16), generator=g, device="cuda").to(torch.int8)[:, :k]
    wscale, bias = torch.rand(70, generator=g, device="cuda") * 1e-3, torch.randn(70, generator=g, device="cuda").to(dtype)
    y = int8.linear(x, weights, wscale, bias)
    check_product(y, *int8.quantize_rows(x), weights, wscale, bias)
