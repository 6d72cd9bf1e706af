"""The block on the gated recurrence in the ways a program uses it: served in 8 bits while its weights change."""
import copy

import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu


def build(width=64, seed=0, dtype=torch.bfloat16):
    torch.manual_seed(seed)
    return vig_b200.GatedRecurrence(width).cuda().to(dtype)


def served(block, x):
    state = torch.zeros(x.shape[0], block.d_inner, device="cuda")
    out, residual = block.step(x, None, state)
    return out, residual, state


@pytest.mark.parametrize("change", ["optimizer", "load_state_dict", "copy_", "to"])
def test_8_bit_steps_follow_the_weights(change):
    """A step behind a change of the weights gives what a block gives that was quantized after it."""
    block, x = build().quantize(), torch.randn(4, 64, device="cuda").bfloat16()
    before = served(block, x)
    if change == "optimizer":
        opt = vig_b200.AdamW(block.parameters(), lr=0.05)
        for p in block.parameters():
            p.grad = torch.ones_like(p)
        opt.step()
    elif change == "load_state_dict":
        block.load_state_dict(build(seed=1).state_dict())
    elif change == "copy_":
        with torch.no_grad():
            block.in_proj.weight.copy_(torch.randn_like(block.in_proj.weight))
    else:
        block.cpu()
        block.in_proj.weight.data.mul_(2)
        block.cuda()
    after = served(block, x)
    fresh = build(seed=2)
    fresh.load_state_dict(block.state_dict())
    want = served(fresh.quantize(), x)
    assert all(torch.equal(a, b) for a, b in zip(after, want))
    assert not torch.equal(after[2], before[2])


def test_8_bit_weights_are_laid_out_once():
    block, x = build().quantize(), torch.randn(1, 64, device="cuda").bfloat16()
    codes = block._codes()[0]
    served(block, x)
    assert block._codes()[0] is codes
    twin = copy.deepcopy(block)
    assert all(torch.equal(a, b) for a, b in zip(served(twin, x), served(block, x)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast(dtype):
    """Three blocks in fp32 under autocast: outputs and gradients of the fp32 run within what 16-bit products and recurrences round (a handful of units
    a block), the residual stream in fp32; and served, with and without 8-bit products."""
    torch.manual_seed(0)
    blocks = torch.nn.ModuleList([vig_b200.GatedRecurrence(64) for _ in range(3)]).cuda()
    x = torch.randn(2, 40, 64, device="cuda")
    unit = 2.0 ** (-8 if dtype == torch.bfloat16 else -11)

    def run():
        h, residual, finals = x, None, []
        for b in blocks:
            h, residual, final = b(h, residual, None, True)
            finals.append(final)
        return h, residual, finals

    want = run()
    w = torch.randn_like(x)
    grads = torch.autograd.grad(((want[0] + want[1]) * w).sum(), list(blocks.parameters()))
    with torch.autocast("cuda", dtype):
        h, residual, finals = run()
    assert h.dtype == dtype and residual.dtype == torch.float32 and all(f.dtype == torch.float32 for f in finals)
    far = lambda a, b: float((a.float() - b).norm() / b.norm())  # noqa: E731
    assert far(h + residual, want[0] + want[1]) < 3 * 8 * unit
    got = torch.autograd.grad(((h + residual) * w).sum(), list(blocks.parameters()))
    assert all(a.dtype == torch.float32 and far(a, b) < 3 * 16 * unit for a, b in zip(got, grads))
    for eight in (False, True):
        if eight:
            for b in blocks:
                b.quantize()
        with torch.no_grad(), torch.autocast("cuda", dtype):
            states = [torch.zeros(2, 64, device="cuda") for _ in blocks]
            for t in range(40):
                h, residual = x[:, t], None
                for b, s in zip(blocks, states):
                    h, residual = b.step(h, residual, s)
        assert far(h + residual, (want[0] + want[1])[:, -1].detach()) < (0.1 if eight else 3 * 8 * unit)


def test_only_16_bits_are_widened():
    block, r = build(dtype=torch.float32), torch.randn(2, 5, 64, device="cuda")
    with pytest.raises(TypeError):
        block(r.double(), r)
    with pytest.raises(TypeError):
        block(r, r.bfloat16())


def test_weights_of_inference_mode():
    """They have no version: quantize() takes them as they are then."""
    with torch.inference_mode():
        block, x = build().quantize(), torch.randn(4, 64, device="cuda").bfloat16()
        before = served(block, x)
        block.in_proj.weight.mul_(2)
        after = served(block.quantize(), x)
        assert not torch.equal(after[2], before[2])
        fresh = build(seed=3)
        fresh.load_state_dict(block.state_dict())
        assert all(torch.equal(a, b) for a, b in zip(after, served(fresh.quantize(), x)))
