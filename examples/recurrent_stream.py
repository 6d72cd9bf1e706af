"""Train a small causal stack of gated-recurrence blocks on a stream of numbers, then serve it one token at a time.

Training: RMS norm behind the residual add and the recurrence with their backward kernels, AdamW with 8-bit states and full-precision copies
of the 16-bit weights.  Serving: 8-bit rows out of the norm into 8-bit products, the recurrence's state updated in place.

    python examples/recurrent_stream.py [--steps 60] [--width 256] [--depth 2] [--length 256] [--batch 16]
"""
import argparse
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import vig_b200  # noqa: E402


class Stream(torch.nn.Module):
    def __init__(self, width, depth):
        super().__init__()
        self.blocks = torch.nn.ModuleList([vig_b200.GatedRecurrence(width) for _ in range(depth)])

    def forward(self, x, states=None):
        """``[B, L, width]`` -> the same, and the states behind the last token."""
        h, residual, finals = x, None, []
        for i, block in enumerate(self.blocks):
            h, residual, final = block(h, residual, states[i] if states else None, True)
            finals.append(final)
        return residual + h, finals

    def step(self, x, states):
        """One token ``[B, width]``; ``states`` are updated in place."""
        h, residual = x, None
        for block, state in zip(self.blocks, states):
            h, residual = block.step(h, residual, state)
        return residual + h


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("steps", 60), ("width", 256), ("depth", 2), ("length", 256), ("batch", 16)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    model = Stream(a.width, a.depth).cuda().bfloat16()
    opt = vig_b200.AdamW(model.parameters(), lr=2e-3, weight_decay=0.01, state_bits=8, master_weights=True)
    gen = torch.Generator(device="cuda").manual_seed(1)
    losses = []
    for _ in range(a.steps):
        x = torch.randn(a.batch, a.length, a.width, generator=gen, device="cuda").bfloat16()
        goal = torch.cumsum(x.float(), 1).roll(1, -1) / 8              # what a state has to hold
        loss = (model(x)[0].float() - goal).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    losses = [float(v) for v in losses]
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps")

    for block in model.blocks:
        block.quantize()
    prefix = a.length - 16
    x = torch.randn(a.batch, a.length, a.width, generator=gen, device="cuda").bfloat16()
    with torch.no_grad():
        whole, _ = model(x)
        _, states = model(x[:, :prefix])
        model.step(x[:, prefix], [s.clone() for s in states])              # the first step loads its kernels
        torch.cuda.synchronize()
        began = time.perf_counter()
        served = torch.stack([model.step(x[:, t], states) for t in range(prefix, a.length)], 1)
        torch.cuda.synchronize()
        took = time.perf_counter() - began
    far = float((served - whole[:, prefix:]).float().norm() / whole[:, prefix:].float().norm())
    print(f"served 16 tokens of {a.batch} streams in {took * 1e3:.2f} ms, {far:.3f} from the whole sequence in 16 bits")
    vig_b200.check_status()
    return losses, far


if __name__ == "__main__":
    main()
