"""A channels-last block of 8-bit token operators: trained for a few steps, then served a token at a time.

    python examples/token_block.py [--steps 50] [--level L3]

The block is a residual feed-forward block over positions (pixels, or tokens): group norm with SiLU, a product in 8-bit integers
to twice the hidden width, a gated SiLU, a product back.  Everything the backward pass needs of the activations is kept as 8-bit
codes; with ``--level L0`` the norm and the gate keep their inputs as they are, for comparison."""
import argparse
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import actnn_b200 as actnn  # noqa: E402


class TokenBlock(nn.Module):
    def __init__(self, channels=256, hidden=512, groups=32):
        super().__init__()
        self.norm = actnn.QGroupNorm(groups, channels, activation="silu")
        self.up = actnn.QInt8Linear(channels, 2 * hidden)
        self.gate = actnn.QGLU("silu")
        self.down = actnn.QInt8Linear(hidden, channels)

    def forward(self, x):                                  # [N, C, H, W], channels last
        tokens = self.norm(x).movedim(1, -1)               # [N, H, W, C]: a position is a row of channels where it lies
        return x + self.down(self.gate(self.up(tokens))).movedim(-1, 1)

    def serve(self, tokens):                               # [T, C] rows that are normalised already
        return self.down(self.gate(self.up(tokens)))


def kept_bytes(model, x):
    """Bytes of activations that the forward pass leaves for the backward pass."""
    def held():
        return torch.cuda.memory_stats()["requested_bytes.all.current"]      # without what the allocator adds to a block

    before = held()
    y = model(x)
    return held() - before - y.numel() * y.element_size()


def train(steps=50, level="L3", device="cuda", dtype=torch.bfloat16, seed=0):
    """Fits a random smooth map of the input; returns the losses, the kept bytes and the model."""
    actnn.set_optimization_level(level)
    torch.manual_seed(seed)
    model = TokenBlock().to(device=device, dtype=dtype).train()
    x = torch.randn(16, 256, 28, 28, device=device, dtype=dtype).contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        target = x + torch.tanh(torch.roll(x, 1, 1)) * 0.5
    optimiser = torch.optim.Adam(model.parameters(), lr=3e-3)
    kept, losses = kept_bytes(model, x), []
    for _ in range(steps):
        loss = (model(x).float() - target.float()).square().mean()
        optimiser.zero_grad(set_to_none=True)
        loss.backward()
        optimiser.step()
        losses.append(loss.detach())
    return [float(v) for v in losses], kept, model


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=50)
    parser.add_argument("--level", default="L3")
    args = parser.parse_args(argv)
    losses, kept, model = train(args.steps, args.level)
    print("loss %.4f -> %.4f over %d steps; %.1f MB of activations kept" % (losses[0], losses[-1], args.steps, kept / 1e6))
    model.eval()
    model.up.freeze(), model.down.freeze()
    with torch.no_grad():
        token = torch.randn(1, 256, device="cuda", dtype=torch.bfloat16)
        print("one token:", tuple(model.serve(token).shape))


if __name__ == "__main__":
    main()
