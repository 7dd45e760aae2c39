"""The token operators together, as examples/token_block.py uses them."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def block():
    spec = importlib.util.spec_from_file_location("token_block", os.path.join(ROOT, "examples", "token_block.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_training_lowers_the_loss_and_keeps_less(cuda_device, block):
    import actnn_b200 as actnn
    losses, kept, _ = block.train(30, "L3")
    assert losses[-1] < 0.7 * losses[0] and all(v == v for v in losses)
    actnn.config.__dict__.update(actnn.conf.QuantizationConfig().__dict__)
    exact, kept_exact, _ = block.train(30, "L0")
    assert abs(losses[-1] - exact[-1]) < 0.05 * exact[0]
    # a byte for each channel that the norm, the products and the gate take, and at most a twentieth of scales, codes of the
    # weights and rounding of the allocator; at L0 the gate's input is kept in 16 bits (the norm's is the caller's own tensor)
    positions = 16 * 28 * 28
    assert positions * 2048 <= kept <= 1.05 * positions * 2048
    assert positions * (256 + 2 * 1024 + 512) <= kept_exact <= 1.05 * positions * (256 + 2 * 1024 + 512)


def test_swapped_activations_give_the_same_steps(cuda_device, block):
    import actnn_b200 as actnn
    here = block.train(4, "L3")[0]
    actnn.config.__dict__.update(actnn.conf.QuantizationConfig().__dict__)
    assert block.train(4, "L4")[0] == here


def test_the_same_steps_twice(cuda_device, block):
    assert block.train(4)[0] == block.train(4)[0]


def test_served_tokens(cuda_device, block):
    model = block.TokenBlock().cuda().half().eval()
    tokens = torch.randn(33, 256, device="cuda").half()
    with torch.no_grad():
        want = model.serve(tokens)
        model.up.freeze(), model.down.freeze()
        assert torch.equal(model.serve(tokens), want)
        for t in (1, 2, 7, 8, 9, 20):                      # every token on its own row, however many come at a time
            assert torch.equal(model.serve(tokens[:t]), want[:t])


def test_command(cuda_device, block, capsys):
    block.main(["--steps", "2"])
    out = capsys.readouterr().out
    assert "loss" in out and "one token: (1, 256)" in out
