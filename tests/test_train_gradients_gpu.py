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


def _calls():
    x, g, s, w = (torch.randn(*shape, device="cuda") for shape in ((2, 5, 64), (2, 5, 64), (2, 64), (64,)))
    return {
        "recurrence": (lambda x, g, s: vig_b200.gated_recurrence(x, g, s, True)[0], (x, g, s)),
        "step": (lambda x, g, s: vig_b200.gated_recurrence_step(x, g, s), (x[:, 0].clone(), g[:, 0].clone(), s)),
        "norm": (lambda x, w, r: vig_b200.add_rmsnorm_train(x, w, r)[0], (x, w, g)),
        "norm_backward": (lambda d, x, w, r, q: vig_b200.add_rmsnorm_backward(d, x, w, 1e-6, r, q)[0], (x, g, w, x + 1, g + 1)),
        "norm8": (lambda x, w, r: vig_b200.add_rmsnorm_8bit(x, w, r)[1], (x, w, g)),
    }


@pytest.mark.parametrize("name,n", [("recurrence", 3), ("step", 3), ("norm", 3), ("norm_backward", 5), ("norm8", 3)])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_refused(name, n, grad_mode):
    """A tangent at any input raises, with or without gradients of reverse mode; a dual level without tangents changes nothing."""
    import torch.autograd.forward_ad as fwad
    call, args = _calls()[name]
    with torch.set_grad_enabled(grad_mode), fwad.dual_level():
        call(*args)
        for i in range(n):
            duals = [fwad.make_dual(t, torch.ones_like(t)) if k == i else t for k, t in enumerate(args)]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(*duals)


@pytest.mark.parametrize("call", [lambda x: vig_b200.gated_recurrence(x, torch.zeros_like(x))[0], lambda x: vig_b200.add_rmsnorm_train(x, torch.ones(64, device="cuda"))[0]],
                         ids=["recurrence", "norm"])
def test_forward_mode_over_the_backward_is_refused(call):
    import torch.autograd.forward_ad as fwad
    x = torch.randn(2, 5, 64, device="cuda", requires_grad=True)
    with fwad.dual_level():
        d = fwad.make_dual(torch.ones(2, 5, 64, device="cuda"), torch.ones(2, 5, 64, device="cuda"))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(call(x), x, d)
