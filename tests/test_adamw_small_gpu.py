"""AdamW where the second moment is below the smallest normal number: its root is not zero, and with a small eps, or none, it is all that the step is
divided by.

Tolerances: v is held in steps of 2^-149, so it is off by up to two of them, its root by half of that part of itself; the rest as in
test_adamw_gpu.py."""
import math

import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu
LR, B1, B2 = 1e-2, 0.9, 0.999


@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-30, 1e-21])
@pytest.mark.parametrize("n", [7, 256, 1000])
def test_subnormal_second_moments(n, eps):
    """Roots of 1e-22 to 1e-19, steps of a size like any other."""
    gen = torch.Generator().manual_seed(n)
    v = 10.0 ** (-43 + 6 * torch.rand(n, generator=gen))
    m = v.double().sqrt().float() * torch.randn(n, generator=gen)
    p, g = torch.randn(n, generator=gen), torch.zeros(n)
    dev = [t.cuda() for t in (p, g, m, v)]
    vig_b200.adamw_step(*[[t] for t in dev], 10, LR, (B1, B2), eps, 0.0)
    v1, m1 = B2 * v.double(), B1 * m.double()
    den = (v1 / (1 - B2 ** 10)).sqrt() + eps
    move = LR / (1 - B1 ** 10) * m1 / den
    off = 2 * 2.0 ** -149 / v1 + 2 * 2.0 ** -149 / m1.abs().clamp_min(1e-45) + 16 * 2.0 ** -24
    assert (v1 < 1.17e-38).sum() > n // 2
    assert ((dev[0].cpu().double() - (p.double() - move)).abs() <= off * move.abs() + 2 * 2.0 ** -24 * (p.abs() + move.abs())).all()


def test_a_root_that_is_not_zero_keeps_its_code():
    """8-bit states of a block whose second moments are all below the smallest normal number."""
    n = 256
    root = torch.linspace(1e-21, 1e-19, n)
    scale = root.max() / 448
    code = (root / scale).to(torch.float8_e4m3fn)
    stood = code.double() * float(scale)
    p, g, m, ms = torch.zeros(n), torch.zeros(n), torch.zeros(n), torch.zeros(1)
    dev = [t.cuda() for t in (p, g, m.to(torch.float8_e4m3fn), code, ms, scale[None])]
    vig_b200.adamw_step([dev[0]], [dev[1]], [dev[2]], [dev[3]], 10, LR, (B1, B2), 1e-25, 0.0, exp_avg_scales=[dev[4]], exp_avg_sq_scales=[dev[5]])
    got = dev[3].cpu().double() * float(dev[5])
    want = stood * math.sqrt(B2)
    # a v of 1e-42 has steps of a thousandth of itself; then half a step of e4m3
    assert (got > 0).all() and ((got - want).abs() <= want / 16 * 1.01 + want * 2e-3 + float(dev[5]) * 2.0 ** -9).all()


def test_zero_stays_zero():
    p, g, m, v = (torch.zeros(300, device="cuda") for _ in range(4))
    vig_b200.adamw_step([p], [g], [m], [v], 3, LR, (B1, B2), 1e-30, 0.0)
    assert all((t == 0).all() for t in (p, m, v))
