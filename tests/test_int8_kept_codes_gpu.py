"""The integer linear layer keeps codes for the gradients that are asked for, and no others."""
import pytest
import torch

from test_int8_linear_gpu import tokens
from test_swap_token_inputs_gpu import held

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("half", ["native", "python"])
@pytest.mark.parametrize("flags", [(True, True, True), (True, False, False), (False, True, False), (False, False, True), (True, False, True)])
def test_bytes(cuda_device, monkeypatch, flags, half):
    from actnn_b200 import _lib, ops
    if half == "python":
        monkeypatch.setattr(_lib, "_native", False)
    t, k, n = 4096, 1024, 512
    x, w, b = tokens(t, k, torch.float16), tokens(n, k, torch.float16, 1), tokens(1, n, torch.float16, 2)[0]
    dy = tokens(t, n, torch.float16, 3)
    every = [v.clone().requires_grad_() for v in (x, w, b)]
    ops.int8_linear.apply(*every).backward(dy)
    mine = [v.requires_grad_(f) for v, f in zip((x, w, b), flags)]

    before = held()
    y = ops.int8_linear.apply(*mine)
    kept = held() - before - y.numel() * 2
    needed = flags[0] * n * (k + 4) + flags[1] * t * (k + 4)
    assert needed <= kept <= needed + 4 * (t + n)       # scales of the other operand at most
    y.backward(dy)
    for got, want, asked in zip(mine, every, flags):
        assert torch.equal(got.grad, want.grad) if asked else got.grad is None
