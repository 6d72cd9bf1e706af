"""States that are infinite: the recurrence's definition, token by token, says which stay infinite, which become NaN and which are untouched."""
import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu


def kind(t):
    """0 finite, 1 inf, 2 -inf, 3 NaN"""
    return torch.isnan(t) * 3 + torch.isposinf(t) * 1 + torch.isneginf(t) * 2


def scan(a, x):
    s, out = torch.zeros_like(x[:, 0]), []
    for t in range(x.shape[1]):
        s = a[:, t] * s + x[:, t]
        out.append(s)
    return torch.stack(out, 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm,reverse", [(0.0, False), (1.0, False), (1.0, True)])
@pytest.mark.parametrize("B,L,D", [(1, 12, 40), (1, 700, 33), (1, 5000, 64), (12, 1500, 96), (64, 400, 768), (30, 400, 1024)])
def test_infinite_states(B, L, D, norm, reverse, dtype):
    """Decays of about a half: over a few hundred tokens their product is 0 in fp32, and an infinity ahead of them has to outlast that; a decay of 0 and an
    infinity of the other sign make it NaN.  The same for the gradients, from the other end."""
    gen = torch.Generator(device="cuda").manual_seed(L)
    x, d_h = (torch.randn(B, L, D, generator=gen, device="cuda").to(dtype) for _ in range(2))
    g = -0.3 - torch.rand(B, L, D, generator=gen, device="cuda")
    g = (torch.log(g.exp() / (1 - g.exp())) if norm else g).to(dtype)
    inf, n = float("inf"), L // 3
    for t in (x, d_h):
        t[:, n, 0], t[:, n, 3] = inf, -inf
        t[:, n, 5], t[:, n + L // 4, 5] = inf, -inf
        t[:, n, 7] = t[:, n, 9] = inf
    g[:, n + L // 4, 7] = -inf                     # a reset of an infinite state
    g[:, 2 * n, 11] = -inf                         # ... and of a finite one
    turn = (lambda t: t.flip(1)) if reverse else (lambda t: t)
    gd = turn(g.double())
    a = torch.sigmoid(gd) if norm else gd.exp()
    leaf = [x.clone().requires_grad_(True), g.clone().requires_grad_(True)]
    h, _ = vig_b200.gated_recurrence(*leaf, reverse=reverse, gate_logit_normalizer=norm)
    assert torch.equal(kind(h.detach()), kind(turn(scan(a, turn(x.double())))))
    dx = torch.autograd.grad(h, leaf[0], d_h)[0]
    later = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    want = scan(later.flip(1), turn(d_h.double()).flip(1)).flip(1)
    assert torch.equal(kind(dx), kind(turn(want)))


def test_infinite_initial_state():
    x, g = torch.randn(2, 3000, 64, device="cuda").bfloat16(), torch.full((2, 3000, 64), -0.5, device="cuda").bfloat16()
    h0 = torch.full((2, 64), float("inf"), device="cuda")
    h, final = vig_b200.gated_recurrence(x, g, h0, True)
    assert torch.isposinf(h).all() and torch.isposinf(final).all()
    g[:, 1000] = float("-inf")
    h, final = vig_b200.gated_recurrence(x, g, h0, True)
    assert torch.isposinf(h[:, :1000]).all() and torch.isnan(h[:, 1000:]).all() and torch.isnan(final).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,D", [(2, 200, 64), (1, 3000, 33), (64, 400, 768)])
def test_what_is_finite_keeps_its_bits(B, L, D, dtype):
    """An infinity changes nothing ahead of itself and in no other channel, forward and in the gradients."""
    gen = torch.Generator(device="cuda").manual_seed(L)
    x, d_h = (torch.randn(B, L, D, generator=gen, device="cuda").to(dtype) for _ in range(2))
    g = (-torch.rand(B, L, D, generator=gen, device="cuda")).to(dtype)

    def run(x, d_h):
        leaf = [x.clone().requires_grad_(True), g.clone().requires_grad_(True)]
        h, final = vig_b200.gated_recurrence(*leaf, None, True)
        return (h.detach(), final.detach(), *torch.autograd.grad(h, leaf, d_h))

    h, final, dx, dg = run(x, d_h)
    n = L // 2
    x2, d2 = x.clone(), d_h.clone()
    x2[:, n, 5], d2[:, n, 9] = float("inf"), float("-inf")
    h2, final2, dx2, dg2 = run(x2, d2)
    assert torch.isposinf(h2[:, n:, 5]).all() and torch.isposinf(final2[:, 5]).all() and torch.isneginf(dx2[:, :n + 1, 9]).all()
    assert not torch.isfinite(dg2[:, n + 1:, 5]).any() and not torch.isfinite(dg2[:, 1:n + 1, 9]).any()
    h2[:, n:, 5], final2[:, 5], dx2[:, :n + 1, 9] = h[:, n:, 5], final[:, 5], dx[:, :n + 1, 9]
    dg2[:, n + 1:, 5], dg2[:, :n + 1, 9] = dg[:, n + 1:, 5], dg[:, :n + 1, 9]
    assert all(torch.equal(a, b) for a, b in zip((h2, final2, dx2, dg2), (h, final, dx, dg)))
