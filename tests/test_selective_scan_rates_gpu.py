"""The selective scan with rates A whose size is past what fp32 can multiply: a state forgets everything at each token, and tokens behind the end of a sequence, or in the part of
a tile of 64 behind its end, leave it as it is."""
import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rate", [float("-inf"), -3e38, -2e38])
@pytest.mark.parametrize("L", [1, 5, 64, 70, 128, 200])
@pytest.mark.parametrize("N", [1, 8, 16, 20])
def test_state_without_memory(N, L, rate):
    """h_t = delta_t u_t B_t: with steps of a power of two and whole numbers all of it is exact."""
    gen = torch.Generator().manual_seed(L + N)
    whole = lambda *s: torch.randint(-4, 5, s, generator=gen).float().cuda()  # noqa: E731
    u, B, C, h0 = whole(3, L, 6), whole(3, L, N), whole(3, L, N), whole(3, 6, N)
    dt, A = torch.full((3, L, 6), 0.5, device="cuda"), torch.full((6, N), rate, device="cuda")
    A[4] = -1.0                                  # a channel that remembers, beside them
    n = torch.tensor([L, max(0, L - 3), 0], device="cuda")
    there = (torch.arange(L, device="cuda") < n[:, None])[..., None]
    for lengths in (None, n):
        y, final = vig_b200.selective_scan(u, dt, A, B, C, initial_state=h0, output_final_state=True, dt_softplus=False, lengths=lengths)
        want = 0.5 * u * (B * C).sum(-1, keepdim=True)
        ends = torch.full((3,), L, device="cuda") if lengths is None else lengths
        last = 0.5 * u[torch.arange(3), ends - 1][..., None] * B[torch.arange(3), ends - 1][:, None]
        last = torch.where((ends > 0)[:, None, None], last, h0)
        if lengths is not None:
            want = torch.where(there, want, torch.zeros_like(want))
        keep = [0, 1, 2, 3, 5]
        assert torch.equal(y[..., keep], want[..., keep]) and torch.equal(final[:, keep], last[:, keep])
        assert torch.isfinite(y).all() and torch.isfinite(final).all()
    state = h0.clone()
    y = vig_b200.selective_scan_step(u[:, 0], dt[:, 0], A, B[:, 0], C[:, 0], state, dt_softplus=False)
    assert torch.equal(state[:, keep], (0.5 * u[:, 0, :, None] * B[:, 0, None])[:, keep]) and torch.isfinite(y).all()


@pytest.mark.parametrize("rate", [float("-inf"), -3e38])
def test_gradients_are_finite(rate):
    """What a state without memory gives back reaches its own token alone; u's and dt's gradients are those of delta u (B . C)."""
    gen = torch.Generator().manual_seed(0)
    whole = lambda *s: torch.randint(-4, 5, s, generator=gen).float().cuda()  # noqa: E731
    u, B, C, d = whole(2, 70, 5), whole(2, 70, 8), whole(2, 70, 8), whole(2, 70, 5)
    dt, A = torch.full((2, 70, 5), 0.5, device="cuda"), torch.full((5, 8), rate, device="cuda")
    leaf = [t.requires_grad_(True) for t in (u, dt, A, B, C)]
    y, _ = vig_b200.selective_scan(*leaf, dt_softplus=False)
    d_u, d_dt, d_A, d_B, d_C = torch.autograd.grad(y, leaf, d)
    with torch.no_grad():
        dot = (B * C).sum(-1, keepdim=True)
        assert torch.equal(d_u, 0.5 * d * dot) and torch.equal(d_dt, d * u * dot) and not d_A.any()
        assert torch.equal(d_B, 0.5 * (d * u).sum(-1, keepdim=True) * C) and torch.equal(d_C, 0.5 * (d * u).sum(-1, keepdim=True) * B)


@pytest.mark.parametrize("L", [3, 64, 70])
def test_rate_of_nan_stays(L):
    t = torch.ones(1, L, 2, device="cuda")
    A = torch.tensor([[float("nan")], [-1.0]], device="cuda")
    with torch.no_grad():
        y, final = vig_b200.selective_scan(t, t, A, t[..., :1], t[..., :1], initial_state=torch.ones(1, 2, 1, device="cuda"), output_final_state=True)
    assert y[..., 0].isnan().all() and final[0, 0].isnan().all() and torch.isfinite(y[..., 1]).all() and torch.isfinite(final[0, 1]).all()
