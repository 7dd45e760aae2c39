"""Norms around a residual branch, gradients of many gates of several rows each: as many gates as rows are gone through at a time, or more, so that
a block (or the blocks that share a row) has whole gates one after another."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CASES = [((64, 8), 16384, "layer", True, 0.1), ((150, 9), 4096, "rms", True, 0.0), ((299, 8), 4097, "layer", True, 0.1), ((2400, 8), 256, "rms", True, 0.1),
         ((40, 11), 20000, "rms", False, 0.0), ((1200, 10), 500, "layer", False, 0.0)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lead,c,kind,post,p", CASES)
def test_gradients(cuda_device, lead, c, kind, post, p, dtype):
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import residual_norm as rn
    from test_residual_norm_gpu import NAMES, Case
    gates, each = lead
    blocks = 1                                                # that share a row: 4096 channels each
    while blocks * 4096 < c:
        blocks *= 2
    threads = 512 if blocks > 1 else (c + 255) // 256 * 32
    assert each >= 8 and gates >= torch.cuda.get_device_properties(0).multi_processor_count * (512 // threads) // blocks
    case = Case(lead, c, (gates, 1), kind, post, p, dtype)
    _, _, (cx, sx, cf, sf), st = rn.run(*case.leaves(), **case.options, codes=True)
    leaves = [None if v is None else v.clone().requires_grad_() for v in case.leaves()]
    asked = [v for v in leaves if v is not None]
    got = torch.autograd.grad(ops.residual_norm.apply(*leaves, **case.options), asked, (case.dr, case.dh))
    given = iter(got)
    grads = [None if v is None else next(given) for v in leaves]
    x, f = case.decoded(cx, sx, case.x), case.decoded(cf, sf, case.branch)
    case.check_gradients(grads, x, f, st)
    # the gate's alone, and all but the gate's: the rows are cut in another way
    only = [v if v is None else v.detach().requires_grad_(n == "gate") for n, v in zip(NAMES, leaves)]
    alone, = torch.autograd.grad(ops.residual_norm.apply(*only, **case.options), [only[-1]], (case.dr, case.dh))
    assert torch.equal(alone, grads[-1])
    rest = [v if v is None else v.detach().requires_grad_(n != "gate") for n, v in zip(NAMES, leaves)]
    asked = [v for v in rest if v is not None and v.requires_grad]
    given = iter(torch.autograd.grad(ops.residual_norm.apply(*rest, **case.options), asked, (case.dr, case.dh)))
    case.check_gradients([next(given) if v is not None and v.requires_grad else None for v in rest], x, f, st)
