"""The selective scan with an infinite step, input or gradient: what the recurrence leaves finite is finite, whatever the number of states (the kernels take them in blocks of 8
and 16), and what it makes infinite is an infinity or a NaN; states themselves are the recurrence's."""
import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu


def make(L, N, dtype, seed):
    """A = -1, steps of 0.1: over 100 tokens an infinite value meets no decay that leaves the type's range.  Maps above 0, so that infinities have one sign."""
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return dict(u=rand(2, L, 5).to(dtype), dt=torch.full((2, L, 5), 0.1).to(dtype), A=-torch.ones(5, N), B=(rand(2, L, N).abs() + 0.1).to(dtype), C=(rand(2, L, N).abs() + 0.1).to(dtype),
                initial_state=rand(2, 5, N))


U = 2.0 ** -24
UNIT = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
INF = float("inf")
others = [0, 2, 4]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 3, 5, 8, 9, 16, 17, 30])
def test_infinite_input(N, dtype):
    t = {k: v.cuda() for k, v in make(100, N, dtype, N).items()}
    with torch.no_grad():
        plain, _ = vig_b200.selective_scan(**t, dt_softplus=False)
        t["u"][:, 20, 1], t["u"][:, 70, 3] = INF, -INF
        y, final = vig_b200.selective_scan(**t, output_final_state=True, dt_softplus=False)
        assert not torch.isfinite(y[:, 20:, 1]).any() and not torch.isfinite(y[:, 70:, 3]).any() and (final[:, 1] == INF).all() and (final[:, 3] == -INF).all()
        assert torch.equal(y[..., others], plain[..., others])
        # ahead of it the same sums, joined in another order: two fp32 evaluations of 20 tokens, each off by at most 2 * 20 (8 + 24 * 0.1 + 4 + N) u of the sum of magnitudes
        mag, _ = vig_b200.selective_scan(**{**t, "u": t["u"].abs(), "initial_state": t["initial_state"].abs()}, dt_softplus=False)
        off, most = (y[:, :20].double() - plain[:, :20].double()).abs(), 80 * (15 + N) * U * mag[:, :20].double() + 2 * UNIT[dtype] * plain[:, :20].double().abs()
        assert (off <= most).all()
        state = t["initial_state"].clone()
        y = vig_b200.selective_scan_step(t["u"][:, 20], t["dt"][:, 20], t["A"], t["B"][:, 20], t["C"][:, 20], state, dt_softplus=False)
        assert not torch.isfinite(y[:, 1]).any() and (state[:, 1] == INF).all() and torch.isfinite(y[:, others]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 3, 5, 8, 9, 16, 17, 30])
def test_infinite_gradient(N, dtype):
    """Without the softplus, where decays may be above 1 and the backward asks what it joins: the infinities of the recurrence."""
    t = {k: v.cuda().requires_grad_(True) for k, v in make(100, N, dtype, N).items()}
    y, _ = vig_b200.selective_scan(**t, dt_softplus=False)
    d = torch.randn(y.shape, generator=torch.Generator().manual_seed(N)).to(dtype).cuda()
    back = lambda: torch.autograd.grad(y, [t["u"], t["initial_state"]], d, retain_graph=True)  # noqa: E731
    plain = back()
    d[:, 40, 1], d[:, 80, 3] = INF, -INF
    d_u, d_0 = back()
    assert (d_u[:, :41, 1] == INF).all() and (d_u[:, :81, 3] == -INF).all() and (d_0[:, 1] == INF).all() and (d_0[:, 3] == -INF).all()
    assert torch.isfinite(d_u[:, 81:]).all() and torch.equal(d_u[..., others], plain[0][..., others]) and torch.equal(d_0[:, others], plain[1][:, others])


@pytest.mark.parametrize("L", [30, 64, 150])
def test_infinite_gradients_stay(L):
    """An infinite gradient at the last token is infinite at the first, and in the state ahead of it, over products of decays (e^-4 a token) that have left the type's range."""
    t = {k: v[:1].cuda() if k not in "A" else v.cuda() for k, v in make(L, 1, torch.float32, 5).items()}
    t["dt"].fill_(4.0)
    leaf = {k: v.requires_grad_(True) for k, v in t.items()}
    y, final = vig_b200.selective_scan(**leaf, output_final_state=True, dt_softplus=False)
    d_y, d_f = torch.zeros_like(y), torch.zeros_like(final)
    d_y[0, -1, 0], d_y[0, -1, 1], d_f[0, 2] = INF, -INF, INF
    d_u, d_0 = torch.autograd.grad([y, final], [leaf["u"], leaf["initial_state"]], [d_y, d_f])
    for got in (d_u[0, 0], d_u[0, L // 2], d_0[0, :, 0]):
        assert got[0] == INF and got[1] == -INF and got[2] == INF and got[3] == 0


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("N", [1, 5, 8, 16, 20])
def test_infinite_step(N, softplus):
    """A step of +inf forgets all before it: the gradients of the tokens ahead are those of a sequence that ends there without a word from behind, and finite."""
    t = {k: v.cuda() for k, v in make(90, N, torch.float32, N).items()}
    t["dt"][:, 50, 2], t["u"][:, 50, 2] = INF, 1.0
    leaf = {k: v.requires_grad_(True) for k, v in t.items()}
    y, final = vig_b200.selective_scan(**leaf, output_final_state=True, dt_softplus=softplus)
    assert not torch.isfinite(y[:, 50:, 2]).any() and (final[:, 2] == INF).all() and torch.isfinite(y[:, :50]).all() and torch.isfinite(y[..., [0, 1, 3, 4]]).all()
    d = torch.randn(y.shape, generator=torch.Generator().manual_seed(0)).cuda()
    d_u, d_dt, d_0 = torch.autograd.grad(y, [leaf["u"], leaf["dt"], leaf["initial_state"]], d, retain_graph=True)
    d[:, 50:, 2] = 0
    short = torch.autograd.grad(y, [leaf["u"], leaf["dt"], leaf["initial_state"]], d)
    for a, b in ((d_u[:, :50], short[0][:, :50]), (d_dt[:, :50], short[1][:, :50]), (d_0, short[2])):
        assert torch.isfinite(a).all() and torch.equal(a, b)
