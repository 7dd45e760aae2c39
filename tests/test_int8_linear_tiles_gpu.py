"""The integer product where a block, or a pair of blocks, computes tile after tile, and where a reduction is shared by two or four
blocks: the cuts that larger layers get, on random codes and against the same product in 64 bits."""
import pytest
import torch

from test_int8_linear_gpu import DTYPES, check_product

pytestmark = pytest.mark.gpu

# (tokens, channels, reduction): what the cut makes of it on 148 SMs
SHARED = [(300, 1000, 2048), (300, 3001, 8192)]                     # by four blocks; by two, whose last channels fill no tile
PAIRS = [(300, 8192, 2048), (512, 3001, 4096),                      # one tile a pair: outputs in boxes; element by element
         (700, 8200, 1700), (1111, 8199, 2100)]                     # several tiles a pair, both kinds of ends in every direction
TILES = [(1100, 8192, 1000), (4000, 5000, 384), (5000, 4100, 200),  # several tiles a block, more stages than a tile fills, or fewer
         (4096, 4099, 300)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,n,k", SHARED + PAIRS + TILES)
def test_product(cuda_device, dtype, t, n, k):
    from actnn_b200.cpp_extension import int8
    g = torch.Generator(device="cuda").manual_seed(t + n + k)
    x = (torch.randn(t, k, generator=g, device="cuda") * torch.exp(torch.randn(t, 1, generator=g, device="cuda"))).to(dtype)
    weights = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    weights[:, :k] = torch.randint(-127, 128, (n, k), generator=g, device="cuda")
    weights, wscale = weights[:, :k], torch.rand(n, generator=g, device="cuda") * 1e-3 + 1e-5
    bias = None if t == 300 else torch.randn(n, generator=g, device="cuda").to(dtype)
    codes, scale = int8.quantize_rows(x)
    y = int8.linear(x, weights, wscale, bias)
    check_product(y, codes, scale, weights, wscale, bias)
    assert torch.equal(int8.matmul(codes, scale, weights, wscale, bias, dtype), y)


@pytest.mark.parametrize("t,n,k", [(300, 3001, 8192), (1111, 8199, 2100), (1100, 8192, 1000)])
def test_the_same_product_many_times(cuda_device, t, n, k):
    """One launch after another on the same codes, two streams at a time: the same bits."""
    from actnn_b200.cpp_extension import int8
    g = torch.Generator(device="cuda").manual_seed(1)
    codes, weights = (int8.quantize_rows(torch.randn(r, k, generator=g, device="cuda")) for r in (t, n))
    want = int8.matmul(*codes, *weights)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got += [int8.matmul(*codes, *weights) for _ in range(8)]
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(v, want) for v in got)
