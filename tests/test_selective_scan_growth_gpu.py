"""The selective scan where states grow (A above 0, or negative steps without the softplus): the runs of tokens that are joined by products of decays have to give what the
recurrence gives token by token.  Reference and bounds are those of the scan's other tests."""
import pytest
import torch

from test_selective_scan_gpu import NAMES, check, compare, make, reference, run

pytestmark = pytest.mark.gpu


def flat(B, L, D, N, dtype, seed):
    """no skip, gate or bias: steps are what stands in dt; A = -1"""
    t = make(B, L, D, N, 0, dtype, seed=seed, z=False, skip=False, bias=False)
    t["A"].fill_(-1.0)
    t["dt"].zero_()
    return t


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("step", [3.0, 3.5])
@pytest.mark.parametrize("first", [0, 5, 40, 64, 100])
def test_growth_that_fades_again(first, step, dtype):
    """Eight tokens by e^3 each (their product, e^24, is past 2^32), tokens that change nothing, eight that fade as much: within a tile and from tile to tile.  L = 150 is two
    whole tiles and a part."""
    t = flat(2, 150, 5, 3, dtype, seed=first)
    t["dt"][:, first:first + 8] = -step
    t["dt"][:, first + 20:first + 28] = step
    compare(t, softplus=False)


def test_growth_by_A():
    """Positive A with the softplus, beside channels that fade."""
    t = flat(1, 90, 6, 5, torch.float32, seed=1)
    t["A"][::2] = 1.0
    t["dt"].fill_(-20.0)
    t["dt"][:, 30:38] = 3.0
    compare(t)


def test_decays_past_the_range_of_nothing():
    """40 tokens by e^3, a product of e^120, over a state of nothing and a gradient of nothing: nothing, and what lies on either side is as it was."""
    t = flat(2, 130, 5, 3, torch.float32, seed=3)
    t["initial_state"].zero_()
    t["u"][:, :60] = 0
    t["dt"][:, 10:50] = -3.0
    t["dt"][:, 60:] = 0.5
    ref, mag, room = reference(t, softplus=False)
    y, final = run(t, softplus=False)
    check(y, ref[0], mag[0], room, ("y", torch.float32))
    check(final, ref[1], mag[1], room, ("final", torch.float32))
    assert not y[:, :60].any()
    # the other way: gradients only in front of the tokens that grow
    t = flat(2, 130, 5, 3, torch.float32, seed=4)
    t["initial_state"].zero_()
    t["u"].zero_()
    t["dt"][:, :30] = 0.5
    t["dt"][:, 40:80] = -3.0
    d_y = torch.randn(2, 130, 5, generator=torch.Generator().manual_seed(0))
    d_y[:, 30:] = 0
    d_f = torch.zeros(2, 5, 3)
    ref, mag, room = reference(t, d_y, d_f, softplus=False)
    for name, o, r, m in zip(("y", "final", *NAMES), run(t, None, d_y, d_f, softplus=False), ref, mag):
        if o is not None:
            check(o, r, m, room, (name, o.dtype))
