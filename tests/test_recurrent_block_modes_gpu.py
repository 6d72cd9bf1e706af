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
