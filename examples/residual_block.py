"""Residual feed-forward blocks in 8-bit floating point: trained for a few steps, then served a token at a time from a captured graph.

    python examples/residual_block.py [--steps 50] [--level L3] [--kind rms]

A block is a product to twice the hidden width, a gated SiLU, dropout and a product back; between two blocks one call normalises the
block's output, drops, gates and adds it to the residual stream, and normalises the stream for the next.  The products run on 8-bit
floating-point codes in both directions, nothing of a dropout is kept, the norms keep 8-bit codes; with ``--level L0`` the norms
and the gated units keep their inputs as they are, for comparison."""
import argparse
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import actnn_b200 as actnn  # noqa: E402


class Block(nn.Module):
    def __init__(self, channels, hidden, kind, p):
        super().__init__()
        self.up = actnn.QFp8Linear(channels, 2 * hidden)
        self.unit = actnn.QGLU("silu")
        self.drop = actnn.QSeededDropout(p)
        self.down = actnn.QFp8Linear(hidden, channels)
        self.norm = actnn.QResidualNorm(channels, kind=kind, gate=0.5, p=p)

    def forward(self, r, h):
        return self.norm(r, self.down(self.drop(self.unit(self.up(h)))))


class Stack(nn.Module):
    def __init__(self, channels=256, hidden=640, blocks=2, kind="rms", p=0.1):
        super().__init__()
        self.blocks = nn.ModuleList(Block(channels, hidden, kind, p) for _ in range(blocks))

    def forward(self, x):                                  # [.., channels]
        r = h = x
        for block in self.blocks:
            r, h = block(r, h)
        return h

    def freeze(self):
        """Codes the weights once, for serving."""
        for block in self.blocks:
            block.up.freeze(), block.down.freeze()
        return self.eval()


def kept_bytes(model, x):
    """Bytes of activations and codes that the forward pass leaves for the backward pass."""
    def held():
        return torch.cuda.memory_stats()["requested_bytes.all.current"]      # without what the allocator adds to a block

    before = held()
    y = model(x)
    return held() - before - y.numel() * y.element_size()


def train(steps=50, level="L3", kind="rms", device="cuda", dtype=torch.bfloat16, seed=0):
    """Fits a random smooth map of the input; returns the losses, the kept bytes and the model."""
    actnn.set_optimization_level(level)
    torch.manual_seed(seed)
    model = Stack(kind=kind).to(device=device, dtype=dtype).train()
    x = torch.randn(8, 500, 256, device=device, dtype=dtype)
    with torch.no_grad():
        target = torch.tanh(torch.roll(x, 1, -1))
    optimiser = torch.optim.Adam(model.parameters(), lr=1e-3)
    kept, losses = kept_bytes(model, x), []
    for _ in range(steps):
        loss = (model(x).float() - target.float()).square().mean()
        optimiser.zero_grad(set_to_none=True)
        loss.backward()
        optimiser.step()
        losses.append(loss.detach())
    return [float(v) for v in losses], kept, model


class Server:
    """A frozen stack captured for a number of tokens."""

    def __init__(self, model, tokens, channels, device="cuda", dtype=torch.bfloat16):
        self.input = torch.zeros(tokens, channels, device=device, dtype=dtype)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.no_grad(), torch.cuda.stream(stream):
            model(self.input)
        torch.cuda.current_stream().wait_stream(stream)
        self.graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(self.graph):
            self.output = model(self.input)

    def __call__(self, tokens):
        self.input.copy_(tokens)
        self.graph.replay()
        return self.output


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=50)
    parser.add_argument("--level", default="L3")
    parser.add_argument("--kind", default="rms", choices=("rms", "layer"))
    args = parser.parse_args(argv)
    losses, kept, model = train(args.steps, args.level, args.kind)
    print("loss %.4f -> %.4f over %d steps; %.1f MB kept" % (losses[0], losses[-1], args.steps, kept / 1e6))
    serve = Server(model.freeze(), 1, 256)
    print("one token:", tuple(serve(torch.randn(1, 256, device="cuda", dtype=torch.bfloat16)).shape))


if __name__ == "__main__":
    main()
