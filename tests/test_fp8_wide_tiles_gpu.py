"""The 8-bit floating-point product's pairs of blocks, wide tiles and reductions shared by two, against the same product in 64 bits: one round of
tiles and several, tokens, channels and reductions that end inside a tile, a pair whose second block has no channels, results that
leave as boxes and ones that do not (tests/test_fp8_cut.py says which kernel takes which sizes)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# tokens, channels, reduction; the kernel and its tile's tokens
PRODUCTS = [((66, 9810, 3466), "pair 96"), ((71, 10176, 3375), "pair 96"), ((4789, 129, 3114), "pair 128"), ((282, 9945, 1921), "pair 128"),
            ((5578, 136, 3134), "pair 128"), ((273, 9560, 2057), "pair 128"), ((139, 9597, 3135), "pair 160"), ((138, 9920, 3354), "pair 160"),
            ((9966, 131, 3034), "pair 192"), ((12825, 258, 1972), "pair 192"), ((9887, 144, 2946), "pair 192"), ((388, 9512, 1999), "pair 192"),
            ((219, 9578, 2968), "pair 224"), ((193, 9752, 2958), "pair 224"),
            ((15432, 138, 1857), "wide 256"), ((12083, 531, 2729), "wide 256"), ((14647, 144, 1961), "wide 256"), ((11599, 520, 3033), "wide 256"),
            ((259, 13178, 1330), "wide 320"), ((14644, 655, 1058), "wide 320"), ((257, 13000, 1460), "wide 320"), ((587, 15544, 1121), "wide 320"),
            ((13096, 266, 3016), "wide 384"), ((646, 14452, 3094), "wide 384"), ((14117, 280, 2959), "wide 384"), ((12897, 792, 3061), "wide 384"),
            ((404, 14821, 385), "wide 448"), ((397, 14270, 576), "wide 448"), ((390, 14375, 648), "wide 448"), ((410, 14547, 773), "wide 448"),
            ((15309, 387, 924), "wide 448"), ((789, 15155, 924), "wide 448"), ((15035, 400, 390), "wide 448"), ((14932, 392, 514), "wide 448"),
            ((419, 14328, 645), "wide 448"), ((385, 14432, 844), "wide 448"), ((15179, 392, 911), "wide 448"), ((1165, 11064, 931), "wide 448"),
            ((33, 4744, 3965), "split2 64"), ((71, 5070, 3999), "split2 96"), ((7283, 64, 5636), "split2 128"), ((130, 6568, 3805), "split2 160"),
            ((9813, 64, 4677), "split2 192"), ((204, 4880, 8090), "split2 224")]


@pytest.mark.parametrize("size,kernel", PRODUCTS, ids=["%s-%dx%dx%d" % (k.replace(" ", ""), *s) for s, k in PRODUCTS])
def test_product(cuda_device, size, kernel):
    from actnn_b200.cpp_extension import fp8
    from test_fp8_linear_gpu import DTYPES, check_product, decoded, tokens
    t, n, k = size
    x, w, b = tokens(t, k, torch.bfloat16), tokens(n, k, torch.bfloat16, 1), tokens(1, n, torch.bfloat16, 2)[0]
    wc, ws = fp8.quantize_weight(w)
    c, s = fp8.quantize(x)
    dx, dw = decoded(c, s), decoded(wc, ws)
    first = fp8.matmul(c, s, wc, ws, b, torch.bfloat16)
    check_product(first, dx, dw, b)
    assert torch.equal(fp8.linear(x, wc, ws, b), first)                # with the codes' launch before it, which it does not wait for
    assert torch.equal(fp8.matmul(c, s, wc, ws, b, torch.bfloat16), first)
    for out in DTYPES:
        check_product(fp8.matmul(c, s, wc, ws, None, out), dx, dw)


def test_nothing_is_written_around_the_results(cuda_device):
    """Results inside a larger buffer: the values before and behind them stay."""
    from actnn_b200 import _lib
    from actnn_b200.cpp_extension import fp8
    from test_fp8_linear_gpu import tokens
    for t, n, k in ((193, 9752, 2958), (219, 9578, 2968), (385, 14432, 844), (404, 14821, 385), (587, 15544, 1121), (71, 5070, 3999)):
        x, w = tokens(t, k, torch.bfloat16), tokens(n, k, torch.bfloat16, 1)
        wc, ws = fp8.quantize_weight(w)
        c, s = fp8.quantize(x)
        want = fp8.matmul(c, s, wc, ws)
        room = torch.full((t * n + 2048,), 7.0, dtype=torch.bfloat16, device="cuda")
        out = room[1024:1024 + t * n]
        _lib.call("actnn_fp8_matmul", out, c.data_ptr(), s.data_ptr(), wc.data_ptr(), ws.data_ptr(), None, out.data_ptr(), t, n, k, c.stride(0), wc.stride(0),
                  _lib.dtype_id(out.dtype), _lib.stream_of(out))
        assert torch.equal(out.view(t, n), want) and bool((room[:1024] == 7).all()) and bool((room[1024 + t * n:] == 7).all())
