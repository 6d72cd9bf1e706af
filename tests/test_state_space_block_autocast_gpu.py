"""The block under autocast, fp32 weights and 16-bit projections, begun from the state that it hands out: token by token, in one piece, and read in and continued."""
import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu


def far(a, b):
    return float((a.detach().double() - b.detach().double()).norm() / b.detach().double().norm())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window", [None, torch.float32, "16 bits"])
def test_state_under_autocast(window, dtype):
    """Every product rounds its operands and its result to 16 bits, five in a row; eight roundings of 2^-8 bound their sum in bf16 (less in fp16)."""
    torch.manual_seed(0)
    block = vig_b200.SelectiveStateSpace(64).cuda()
    x = torch.randn(2, 40, 64, device="cuda")
    with torch.no_grad():
        whole, _, _ = block(x)
        with torch.autocast("cuda", dtype=dtype):
            plain, _, _ = block(x)
            begin = lambda: block.empty_state(2, dtype=dtype if window == "16 bits" else window)  # noqa: E731
            state = begin()
            outs = [block.step(x[:, i], None, state)[0] for i in range(40)]
            y, r, state2 = block(x[:, :30], None, begin(), output_final_state=True)
            rest = [block.step(x[:, i], None, state2)[0] for i in range(30, 40)]
            again, _, _ = block(x, None, begin())
    assert plain.dtype == y.dtype == again.dtype == outs[0].dtype == rest[0].dtype == dtype and state2[0].dtype == state[0].dtype
    assert torch.equal(state2[1].isfinite().all(), torch.tensor(True, device="cuda"))
    for got in (torch.stack(outs, 1), torch.cat([y, torch.stack(rest, 1)], 1), again, plain):
        assert far(got, whole) < 3e-2
    # a window of zeros is none, and the convolution rounds its sums to 16 bits once whatever the window's type
    assert torch.equal(again, plain)


def test_gradients_from_a_given_state():
    torch.manual_seed(1)
    block = vig_b200.SelectiveStateSpace(32).cuda()
    x = torch.randn(2, 12, 32, device="cuda")
    state = block.empty_state(2)
    grads = []
    for s in (None, state):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y, _, _ = block(x, None, s)
        grads.append(torch.autograd.grad(y.float().square().sum(), list(block.parameters())))
    # the widened call gives the convolution's gradients back rounded to 16 bits once, the other in 16 bits: the same values
    for a, b in zip(*grads):
        assert torch.isfinite(a).all() and far(a, b) < 3e-2


def test_types_that_would_lose():
    """A 16-bit window with fp32 tokens is refused: it cannot take them up."""
    block = vig_b200.SelectiveStateSpace(32).cuda()
    with pytest.raises(TypeError):
        block.step(torch.randn(2, 32, device="cuda"), None, block.empty_state(2, dtype=torch.bfloat16))
