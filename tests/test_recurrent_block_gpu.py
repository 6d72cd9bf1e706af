"""The causal block on the gated recurrence: trained with AdamW, then served token by token."""
import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu


def build(dtype, width=64, depth=2, seed=0):
    torch.manual_seed(seed)
    return torch.nn.ModuleList([vig_b200.GatedRecurrence(width) for _ in range(depth)]).cuda().to(dtype)


def forward(blocks, x, states=None):
    h, residual, finals = x, None, []
    for i, b in enumerate(blocks):
        h, residual, final = b(h, residual, states[i] if states else None, True)
        finals.append(final)
    return residual + h, finals


def plain(block, hidden, residual):
    """The block's formula in 64 bits"""
    r = hidden if residual is None else hidden + residual
    y = r * (r.square().mean(-1, keepdim=True) + block.norm.eps).rsqrt() * block.norm.weight.double()
    x, g, o = (y @ block.in_proj.weight.double().t()).chunk(3, -1)
    a = (torch.nn.functional.logsigmoid(g) / block.gate_logit_normalizer).exp()
    s, hs = torch.zeros_like(x[:, 0]), []
    for t in range(x.shape[1]):
        s = a[:, t] * s + x[:, t]
        hs.append(s)
    return (torch.stack(hs, 1) * torch.nn.functional.silu(o)) @ block.out_proj.weight.double().t(), r


def test_block_and_gradients_against_the_formula():
    blocks = build(torch.float32)
    x = torch.randn(2, 37, 64, device="cuda")
    out, _ = forward(blocks, x)
    h, residual = x.double(), None
    for b in blocks:
        h, residual = plain(b, h, residual)
    ref = h + residual
    # fp32 throughout, products by the library in fp32 (no tf32): sums of 64 to 192 terms, 37 steps, two blocks
    assert float((out.double() - ref).abs().max() / ref.abs().max()) < 1e-5
    w = torch.randn_like(out)
    got = torch.autograd.grad((out * w).sum(), list(blocks.parameters()))
    want = torch.autograd.grad((ref * w.double()).sum(), list(blocks.parameters()))
    for a, b in zip(got, want):
        assert float((a.double() - b.double()).norm() / b.double().norm()) < 1e-5


def test_training_and_serving():
    """Train on sequences whose next value depends on a running sum; a prefix and single tokens then give what the whole sequence gave."""
    blocks = build(torch.bfloat16, width=128)
    opt = vig_b200.AdamW(blocks.parameters(), lr=3e-3, weight_decay=0.0, master_weights=True, state_bits=8)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(8, 96, 128, generator=gen, device="cuda").bfloat16()
    goal = torch.cumsum(x.float(), 1).roll(1, -1) / 8
    losses = []
    for _ in range(40):
        out, _ = forward(blocks, x)
        loss = (out.float() - goal).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < 0.7 * losses[0]
    with torch.no_grad():
        whole, _ = forward(blocks, x)
        out, states = forward(blocks, x[:, :90])
        for quantized in (False, True):
            if quantized:
                for b in blocks:
                    b.quantize()
            live = [s.clone() for s in states]
            for t in range(90, 96):
                h, residual = x[:, t], None
                for b, s in zip(blocks, live):
                    h, residual = b.step(h, residual, s)
                err = float((residual + h - whole[:, t]).float().norm() / whole[:, t].float().norm())
                # 16 bits: a handful of roundings of 2^-9 a block; 8-bit products: codes of 1/16, averaged over 128 terms, three projections wide
                assert err < (0.1 if quantized else 0.02), (quantized, t, err)


def test_example_runs():
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import recurrent_stream
    losses, far = recurrent_stream.main(["--steps", "30", "--width", "64", "--length", "48", "--batch", "4"])
    # the loss falls; 8-bit products against 16-bit ones as above
    assert losses[-1] < losses[0] and far < 0.1
