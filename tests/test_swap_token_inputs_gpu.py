"""At level "swap" nothing is compressed and what the backward pass needs waits in host memory: the inputs of the activations and of
the norm, too."""
import gc

import pytest
import torch

from test_group_norm_gpu import data, last, parameters

pytestmark = pytest.mark.gpu


def held():
    gc.collect()
    torch.cuda.synchronize()
    torch.empty(1, device="cuda")                        # the allocator takes back what copies on other streams have finished with
    return torch.cuda.memory_stats()["requested_bytes.all.current"]


def run(call, leaves, dy):
    """Bytes that the forward pass leaves on the GPU besides its output and the caller's tensors; output and gradients."""
    leaves = [v.clone(memory_format=torch.preserve_format).requires_grad_() for v in leaves]
    grads = [None] * len(leaves)
    for i, v in enumerate(leaves):
        v.register_hook(lambda g, i=i: grads.__setitem__(i, g))
    before = held()
    h = leaves[0] * 1                                    # an intermediate tensor that only the operator can keep alive
    y = call(h, *leaves[1:])
    del h
    kept = held() - before - y.numel() * y.element_size()
    y.backward(dy)
    return kept, [y.detach()] + grads


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_inputs_leave_the_gpu(cuda_device, dtype):
    import actnn_b200 as actnn
    from actnn_b200 import ops
    shape = (8, 64, 32, 32)
    x, (w, b) = last(data(shape, dtype)), parameters(64)
    calls = [(lambda v: ops.activation.apply(v, "gelu"), [x], last(data(shape, dtype, 1))),
             (lambda v: ops.glu.apply(v, "silu"), [x], data((8, 64, 32, 16), dtype, 1)),
             (lambda v, p, q: ops.group_norm.apply(v, 8, p, q, 1e-5, "silu"), [x, w, b], last(data(shape, dtype, 1)))]
    for call, leaves, dy in calls:
        actnn.config.__dict__.update(actnn.conf.QuantizationConfig().__dict__)
        actnn.set_optimization_level("L0")
        here, want = run(call, leaves, dy)
        actnn.set_optimization_level("swap")
        run(call, leaves, dy)                             # the first call makes the workspace that later ones share
        parked, got = run(call, leaves, dy)
        size = x.numel() * x.element_size()
        assert here >= size and parked < size // 16
        assert all(torch.equal(g, v) for g, v in zip(got, want))
