"""How far the selective scan's sums over long sequences are from 64 bits, beside the recurrence evaluated token by token in fp32 with torch."""
import math

import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu


def recurrence(t, d_y, dtype):
    """y and the gradients of all inputs, token by token"""
    u, dt, A, B, C = leaf = [v.to(dtype).requires_grad_(True) for v in t]
    h, ys = torch.zeros(u.shape[0], u.shape[2], A.shape[1], dtype=dtype, device=u.device), []
    for i in range(u.shape[1]):
        h = torch.exp(dt[:, i, :, None] * A) * h + (dt[:, i] * u[:, i])[..., None] * B[:, i, None]
        ys.append((h * C[:, i, None]).sum(-1))
    y = torch.stack(ys, 1)
    return [y.detach(), *torch.autograd.grad(y, leaf, d_y.to(dtype))]


@pytest.mark.parametrize("B,L,D", [(8, 1024, 64), (2, 2048, 128)])
def test_beside_fp32(B, L, D):
    """Steps from a thousandth to a tenth, rates 1 to 16, as such a layer begins.  Errors of a decay that have one sign add up over the tokens that a state remembers.  expf is off by
    up to 1 ulp, 2 u, of both signs; the kernel's decay has a mean error of 0.3 u at most over such arguments (the bound 2 leaves as much again as fp32's own errors)."""
    gen = torch.Generator(device="cuda").manual_seed(L)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    dt = torch.exp(torch.rand(B, L, D, generator=gen, device="cuda") * math.log(4) + torch.rand(D, generator=gen, device="cuda") * math.log(25) + math.log(1e-3))
    t = [rand(B, L, D), dt, -torch.arange(1.0, 17.0, device="cuda").repeat(D, 1) * (1 + 0.1 * rand(D, 16)), rand(B, L, 16), rand(B, L, 16)]
    d_y = rand(B, L, D)
    exact, fp32 = recurrence(t, d_y, torch.float64), recurrence(t, d_y, torch.float32)
    leaf = [v.clone().requires_grad_(True) for v in t]
    y, _ = vig_b200.selective_scan(*leaf, dt_softplus=False)
    ours = [y.detach(), *torch.autograd.grad(y, leaf, d_y)]
    far = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    for name, o, f, e in zip(("y", "u", "dt", "A", "B", "C"), ours, fp32, exact):
        assert far(o, e) <= 2 * far(f, e), f"{name}: {far(o, e):.2e} where fp32 is {far(f, e):.2e}"
