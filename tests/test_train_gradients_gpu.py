"""What the operators of a trained and served recurrent block do where a gradient is asked for that they do not have: they refuse."""
import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["x", "weight", "residual"])
@pytest.mark.parametrize("prenorm", [False, True])
def test_8_bit_rows_do_not_cut_a_graph(which, prenorm):
    """The codes have no gradient, and the sum that comes with them would be without the gradient of what is before it."""
    t = dict(x=torch.randn(3, 64, device="cuda"), weight=torch.ones(64, device="cuda"), residual=torch.randn(3, 64, device="cuda"))
    want = vig_b200.add_rmsnorm_8bit(**t, prenorm=prenorm)
    t[which].requires_grad_(True)
    with pytest.raises(NotImplementedError, match="no gradient"):
        vig_b200.add_rmsnorm_8bit(**t, prenorm=prenorm)
    with torch.no_grad():
        got = vig_b200.add_rmsnorm_8bit(**t, prenorm=prenorm)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
