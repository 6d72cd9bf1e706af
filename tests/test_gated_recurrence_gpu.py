"""The gated recurrence against its definition in 64 bits, token by token.

Tolerances come from a running error analysis: with u = 2^-24, every fp32 step of h = a h + x adds at most 4 u of the sum of magnitudes S
(a rounding of the product, of the sum, and as many again where a chunk's share is joined), and a decay that is off by E of itself adds
E a S.  Both are carried along by the same recurrence.  The outputs are rounded once more to their type."""
import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
UNIT = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # half a unit in the last place, with room for one tie
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}


def decay(g, norm):
    return (torch.nn.functional.logsigmoid(g) / norm).exp() if norm else g.exp()


def decay_error(g, norm, dtype):
    """Relative error of an fp32 decay: exp is right to 2 ulp, its argument to a few u of itself, and with raw logits of 16 bits a logarithm that
    is right to 2^-20 absolute stands in its place."""
    if not norm:
        return 8 * U + 2 * U * g.abs().clamp_max(200)
    ls = torch.nn.functional.logsigmoid(g).abs() / norm
    return 8 * U + (4 * U if dtype == torch.float32 else 2.0 ** -20) * (ls.clamp_max(200) + (0 if dtype == torch.float32 else 1 / norm))


def scan(a, x, s, err_in=None, err0=0.0, ea=None):
    """(states before, states after, bound of their error) of s = a s + x along dim 1"""
    before, after, bound = [], [], []
    mag, err = s.abs(), torch.zeros_like(s) + err0
    for t in range(x.shape[1]):
        before.append(s)
        err = a[:, t] * err + ea[:, t] * a[:, t] * mag
        mag = a[:, t] * mag + x[:, t].abs()
        err = err + 4 * U * mag + (0 if err_in is None else err_in[:, t])
        s = a[:, t] * s + x[:, t]
        after.append(s)
        bound.append(err)
    stack = lambda v, like: torch.stack(v, 1) if v else like  # noqa: E731
    return stack(before, x), stack(after, x), stack(bound, x), s, err


def make(B, L, D, dtype, norm, seed, state=True, gates=None):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(B, L, D, generator=gen).to(dtype)
    g = torch.randn(B, L, D, generator=gen)
    g = (g * 2 if norm else -torch.rand(B, L, D, generator=gen) * 0.3 if gates is None else gates(g)).to(dtype)
    h0 = torch.randn(B, D, generator=gen) if state else None
    return x, g, h0


def check(got, ref, bound, dtype):
    got = got.double().cpu()
    off = (got - ref).abs()
    most = bound + UNIT[dtype] * (ref.abs() + bound) + TINY[dtype]
    assert torch.isfinite(got).all()
    assert (off <= most).all(), f"worst {float((off / most).max()):.2f} of the bound"


def reference(x, g, h0, norm, reverse, dtype):
    turn = (lambda t: t.flip(1)) if reverse else (lambda t: t)
    xd, gd = turn(x.double()), turn(g.double())
    a, ea = decay(gd, norm), decay_error(gd, norm, dtype)
    s = torch.zeros(x.shape[0], x.shape[2], dtype=torch.float64) if h0 is None else h0.double()
    before, h, eh, final, ef = scan(a, xd, s, ea=ea)
    return turn, gd, a, ea, before, h, eh, final, ef


SHAPES = [(1, 1, 1), (2, 1, 64), (1, 2, 33), (3, 7, 5), (2, 65, 64), (1, 128, 192), (2, 129, 193), (1, 511, 96), (1, 1021, 40), (1, 2049, 8), (5, 300, 130)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm,reverse", [(0.0, False), (16.0, False), (1.0, True), (0.0, True)])
@pytest.mark.parametrize("B,L,D", SHAPES)
def test_forward_and_gradients(B, L, D, norm, reverse, dtype):
    x, g, h0 = make(B, L, D, dtype, norm, seed=L + D, state=(L + D) % 3 != 0)
    turn, gd, a, ea, before, h, eh, final, ef = reference(x, g, h0, norm, reverse, dtype)
    leaf = [t.cuda().requires_grad_(True) for t in (x, g, h0) if t is not None]
    got, got_final = vig_b200.gated_recurrence(leaf[0], leaf[1], leaf[2] if h0 is not None else None, True, reverse=reverse, gate_logit_normalizer=norm)
    check(got, turn(h), turn(eh), dtype)
    check(got_final, final, ef, torch.float32)

    gen = torch.Generator().manual_seed(7)
    d_h, d_f = torch.randn(B, L, D, generator=gen).to(dtype), torch.randn(B, D, generator=gen)
    grads = torch.autograd.grad([got, got_final], leaf, [d_h.cuda(), d_f.cuda()])
    # u_t = a_t (dh_t + u_{t+1}); dx_t = dh_t + u_{t+1}, carried as d_x_t = dh_t + a_{t+1} d_x_{t+1}
    later = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1).flip(1)
    elater = torch.cat([ea[:, 1:], torch.zeros_like(a[:, :1])], 1).flip(1)
    _, dx, edx, _, _ = scan(later, turn(d_h.double()).flip(1), d_f.double(), ea=elater)
    dx, edx = dx.flip(1), edx.flip(1)
    u, eu = a * dx, a * edx + (ea + 2 * U) * a * dx.abs()
    # the backward reads h as it was rounded
    ebefore = torch.cat([torch.zeros_like(eh[:, :1]), eh[:, :-1] + UNIT[dtype] * (h[:, :-1].abs() + eh[:, :-1]) + TINY[dtype]], 1)
    dg = u * before
    edg = eu * before.abs() + u.abs() * ebefore + eu * ebefore + 4 * U * dg.abs()
    if norm:
        s = torch.sigmoid(-gd) / norm
        dg, edg = dg * s, edg * s + dg.abs() * s * 16 * U
    check(grads[0], turn(dx), turn(edx), dtype)
    check(grads[1], turn(dg), turn(edg), dtype)
    if h0 is not None:
        check(grads[2], u[:, 0], eu[:, 0], torch.float32)


@pytest.mark.parametrize("B,L,D,dtype", [(1, 16384, 96, torch.bfloat16), (2, 5000, 200, torch.float32), (40, 260, 1024, torch.float16), (300, 3, 2000, torch.bfloat16),
                                         (64, 4096, 70, torch.bfloat16)])
def test_long_and_wide(B, L, D, dtype):
    """Sizes at which the sequence is cut among many blocks, and at which it is not; the first and last entries against 64 bits."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, g = (torch.randn(B, L, D, generator=gen, device="cuda").to(dtype) for _ in range(2))
    h, final = vig_b200.gated_recurrence(x, g, None, True, gate_logit_normalizer=16.0)
    for b in {0, B - 1}:
        _, _, _, _, _, ref, eh, rf, ef = reference(x[b:b + 1].cpu(), g[b:b + 1].cpu(), None, 16.0, False, dtype)
        check(h[b:b + 1], ref, eh, dtype)
        check(final[b:b + 1], rf, ef, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L", [5, 300])
def test_strides_and_offsets(dtype, L):
    """Column slices of a wider projection, rows that begin off 4 bytes, a transposed batch, a state that is expanded: same numbers as from copies."""
    wide = torch.randn(L, 3, 3 * 97 + 1, generator=torch.Generator().manual_seed(1)).to(dtype).cuda().transpose(0, 1)
    x, g = wide[..., 1:98], wide[..., 98:195]
    h0 = torch.randn(1, 97, device="cuda").expand(3, 97)
    got = vig_b200.gated_recurrence(x, g, h0, True, gate_logit_normalizer=16.0)
    ref = vig_b200.gated_recurrence(x.contiguous(), g.contiguous(), h0.contiguous(), True, gate_logit_normalizer=16.0)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_prefix_and_steps_are_the_whole_sequence(dtype):
    """A prefix, a chunk of new tokens and single tokens, each continued from the state before, give what one call over all gives."""
    x, g, h0 = (t.cuda() for t in make(3, 40, 70, dtype, 1.0, seed=5))
    kw = dict(gate_logit_normalizer=1.0)
    whole, final = vig_b200.gated_recurrence(x, g, h0, True, **kw)
    h1, s = vig_b200.gated_recurrence(x[:, :21], g[:, :21], h0, True, **kw)
    h2, s = vig_b200.gated_recurrence(x[:, 21:30], g[:, 21:30], s, True, **kw)
    table = torch.full((3, 100), 7.0, device="cuda")
    state = table[:, 11:81]
    state.copy_(s)
    steps = [vig_b200.gated_recurrence_step(x[:, t], g[:, t], state, **kw) for t in range(30, 40)]
    got = torch.cat([h1, h2, torch.stack(steps, 1)], 1)
    # an association of the same sums: each within the bound of one call
    _, _, _, _, _, ref, eh, rf, ef = reference(x.cpu(), g.cpu(), h0.cpu(), 1.0, False, dtype)
    check(got, ref, eh, dtype)
    check(state, rf, ef, torch.float32)
    assert (table[:, :11] == 7).all() and (table[:, 81:] == 7).all()


@pytest.mark.parametrize("B,D,dtype", [(1, 1, torch.float32), (8, 768, torch.bfloat16), (3, 193, torch.float16), (700, 1000, torch.bfloat16), (257, 516, torch.float32)])
@pytest.mark.parametrize("norm", [0.0, 1.0])
def test_step(B, D, dtype, norm):
    x, g, h0 = make(B, 1, D, dtype, norm, seed=B + D)
    _, _, _, _, _, ref, eh, rf, ef = reference(x, g, h0, norm, False, dtype)
    state = h0.cuda()
    before = state._version
    h = vig_b200.gated_recurrence_step(x[:, 0].cuda(), g[:, 0].cuda(), state, gate_logit_normalizer=norm)
    check(h, ref[:, 0], eh[:, 0], dtype)
    check(state, rf, ef, torch.float32)
    assert state._version > before


@pytest.mark.parametrize("L", [6, 400])
def test_resets_and_masked_tokens(L):
    """A log-gate of -inf starts the state anew whatever it held (of finite values); log-gate 0 with x = 0 passes it on unchanged; the lowest
    finite gate is a reset too."""
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(2, L, 48, generator=gen)
    g = -torch.rand(2, L, 48, generator=gen)
    g[:, L // 2] = float("-inf")
    g[:, L // 3] = torch.finfo(torch.float32).min
    x[:, L - 2:], g[:, L - 2:] = 0, 0
    h, final = vig_b200.gated_recurrence(x.cuda(), g.cuda(), torch.full((2, 48), 1e30, device="cuda"), True)
    h = h.cpu()
    assert torch.equal(h[:, L // 2], x[:, L // 2]) and torch.equal(h[:, L // 3], x[:, L // 3])
    assert torch.equal(h[:, L - 2], h[:, L - 3]) and torch.equal(h[:, L - 1], h[:, L - 3]) and torch.equal(final.cpu(), h[:, L - 1])
    xg, gg = x.cuda().requires_grad_(True), g.cuda().requires_grad_(True)
    out, _ = vig_b200.gated_recurrence(xg, gg)
    dx, dg = torch.autograd.grad(out, (xg, gg), torch.ones_like(out))
    assert torch.isfinite(dx).all() and torch.isfinite(dg).all() and (dg[:, L // 2] == 0).all()


def test_growing_gates_from_an_empty_state():
    """Decays above one over a whole chunk: products of them overflow where the state is 0 and must not reach it."""
    x, g = torch.zeros(1, 600, 64, device="cuda"), torch.full((1, 600, 64), 3.0, device="cuda")
    x[:, 590:] = 1
    h, final = vig_b200.gated_recurrence(x, g, None, True)
    assert (h[:, :590] == 0).all() and torch.isfinite(h).all()
    ref = sum(torch.e ** (3.0 * k) for k in range(10))
    assert float((final / ref - 1).abs().max()) < 10 * (8 * U + 6 * U) + 40 * U
    d = torch.autograd.grad(vig_b200.gated_recurrence(x.requires_grad_(True), g)[0][:, 590:].sum(), x)[0]
    assert not torch.isnan(d).any()


def test_nan_and_infinity_stay_in_their_channel():
    x, g = torch.randn(2, 200, 64, device="cuda"), -torch.rand(2, 200, 64, device="cuda")
    clean = vig_b200.gated_recurrence(x, g)[0]
    x[0, 50, 3], x[1, 60, 5] = float("nan"), float("inf")
    got = vig_b200.gated_recurrence(x, g)[0]
    assert torch.isnan(got[0, 50:, 3]).all() and not torch.isfinite(got[1, 60:, 5]).any()
    got[0, 50:, 3], got[1, 60:, 5] = clean[0, 50:, 3], clean[1, 60:, 5]
    assert torch.equal(got, clean)


def test_gradients_against_differences():
    """The formula of the gradients against central differences of the call itself, in fp32 along random directions."""
    x, g, h0 = (t.cuda().requires_grad_(True) for t in make(2, 70, 33, torch.float32, 1.0, seed=9))
    w, wf = torch.randn(2, 70, 33, device="cuda"), torch.randn(2, 33, device="cuda")

    def value(*ins):
        h, f = vig_b200.gated_recurrence(*ins, True, gate_logit_normalizer=1.0)
        return (h.double() * w).sum() + (f.double() * wf).sum()

    for t, grad in zip((0, 1, 2), torch.autograd.grad(value(x, g, h0), (x, g, h0))):
        ins = [x.detach(), g.detach(), h0.detach()]
        v = torch.randn_like(ins[t])
        eps = 2.0 ** -7
        ends = []
        for sign in (1, -1):
            moved = list(ins)
            moved[t] = ins[t] + sign * eps * v
            ends.append(float(value(*moved)))
        diff, want = (ends[0] - ends[1]) / (2 * eps), float((grad.double() * v).sum())
        # x and h0 enter linearly: rounding only, 2 U of the sum of magnitudes over the step; g by eps^2 / 6 of the third derivative on top
        size = float((grad.double() * v).abs().sum())
        assert abs(diff - want) <= (2.0 ** -12 + (eps ** 2 * 16 if t == 1 else 0)) * size


def test_same_bits_twice_and_on_another_stream():
    x, g, h0 = (t.cuda() for t in make(2, 3000, 192, torch.bfloat16, 16.0, seed=4))
    a, fa = vig_b200.gated_recurrence(x, g, h0, True, gate_logit_normalizer=16.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b, fb = vig_b200.gated_recurrence(x, g, h0, True, gate_logit_normalizer=16.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b) and torch.equal(fa, fb)


def test_replays_in_a_graph():
    x, g, h0 = (t.cuda() for t in make(2, 500, 96, torch.float16, 1.0, seed=6))
    vig_b200.gated_recurrence(x, g, h0, True, gate_logit_normalizer=1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, f = vig_b200.gated_recurrence(x, g, h0, True, gate_logit_normalizer=1.0)
    x.copy_(torch.randn_like(x))
    graph.replay()
    ref, rf = vig_b200.gated_recurrence(x, g, h0, True, gate_logit_normalizer=1.0)
    assert torch.equal(h, ref) and torch.equal(f, rf)


@pytest.mark.parametrize("B,L,D", [(0, 4, 8), (2, 0, 8), (2, 4, 0)])
def test_nothing_to_do(B, L, D):
    x, h0 = torch.zeros(B, L, D, device="cuda", requires_grad=True), torch.randn(B, D, device="cuda", requires_grad=True)
    h, f = vig_b200.gated_recurrence(x, x.detach(), h0, True)
    assert h.shape == (B, L, D) and f.shape == (B, D)
    if L == 0:
        assert torch.equal(f, h0)
        assert torch.equal(vig_b200.gated_recurrence(x.detach(), x.detach(), None, True)[1], torch.zeros_like(f))
    gx, g0 = torch.autograd.grad(h.sum() + (2 * f).sum(), (x, h0))
    assert gx.shape == x.shape and g0.shape == h0.shape and (L or torch.equal(g0, torch.full_like(g0, 2.0)))


def test_refusals():
    x, s = torch.zeros(2, 4, 8, device="cuda"), torch.zeros(2, 8, device="cuda")
    call = vig_b200.gated_recurrence
    for bad in (lambda: call(x, x[:, :3]), lambda: call(x[0], x[0]), lambda: call(x, x, s[:1]), lambda: call(x.transpose(1, 2), x.transpose(1, 2)),
                lambda: call(x, x, s, gate_logit_normalizer=-1.0), lambda: call(x, x, s, gate_logit_normalizer=float("nan")),
                lambda: vig_b200.gated_recurrence_step(x[:, 0], x[:, 0], s[:1].expand(2, 8)), lambda: vig_b200.gated_recurrence_step(x, x, s)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: call(x, x.half()), lambda: call(x.double(), x.double()), lambda: call(x, x, s.half()), lambda: call(x.int(), x.int()), lambda: call(x, None)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: call(x.cpu(), x), lambda: call(x, x.cpu()), lambda: call(x, x, s.cpu())):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(NotImplementedError):
        vig_b200.gated_recurrence_step(x[:, 0].clone().requires_grad_(True), x[:, 0], s)
    leaf = x.clone().requires_grad_(True)
    (g1,) = torch.autograd.grad(call(leaf, x)[0].square().sum(), leaf, create_graph=False)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(call(leaf, x)[0].square().sum(), leaf, create_graph=True)


def test_c_entry_refuses_before_any_launch():
    from vig_b200 import _lib
    L_ = _lib.lib()
    fwd = lambda B=1, L=4, D=8, norm=0.0, dtype=0, ptr=None: L_.vig_gated_recurrence_fwd(ptr, ptr, None, 0, ptr, None, 0, B, L, D, None, None, None, norm, 0, dtype, None, None)  # noqa: E731
    assert fwd() == -1 and fwd(dtype=3) == -3 and fwd(B=-1) == -2 and fwd(norm=-1.0) == -6 and fwd(norm=float("nan")) == -6 and fwd(L=0) == 0
    assert L_.vig_gated_recurrence_bwd(None, None, None, None, None, None, None, None, 1, 4, 8, None, None, None, 0.0, 0, 0, None, None) == -1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("L", [5, 90])
def test_masked_logits(L, dtype):
    """Raw logits of -inf or the type's lowest value shut the state out, +inf and the highest keep it whole; gradients there are 0 and the
    others what they are without them."""
    x, g, _ = make(2, L, 24, dtype, 16.0, seed=12, state=False)
    shut, keep = L // 2, L // 3
    g[0, shut], g[1, shut] = float("-inf"), torch.finfo(dtype).min
    g[0, keep], g[1, keep] = float("inf"), torch.finfo(dtype).max
    leaf = [x.cuda().requires_grad_(True), g.cuda().requires_grad_(True)]
    h, _ = vig_b200.gated_recurrence(*leaf, gate_logit_normalizer=16.0)
    dx, dg = torch.autograd.grad(h, leaf, torch.ones_like(h))
    h, dx, dg = h.detach().cpu(), dx.cpu(), dg.cpu()
    assert torch.isfinite(h).all() and torch.isfinite(dx).all() and torch.isfinite(dg).all()
    # sigmoid(lowest fp16)^(1/16) = e^-4094 and less: nothing of the state before is left
    assert torch.equal(h[:, shut], x[:, shut]) and (dg[:, shut] == 0).all() and (dg[:, keep] == 0).all()
    ref = h.float()[:, keep - 1] + x.float()[:, keep]
    off = (h.float()[:, keep] - ref).abs()
    assert (off <= 3 * UNIT[dtype] * (ref.abs() + h.float()[:, keep - 1].abs())).all()


def test_no_token_hands_on_any_state():
    x = torch.zeros(3, 0, 20, device="cuda")
    for h0 in (torch.randn(1, 20, device="cuda").expand(3, 20), torch.randn(3, 50, device="cuda")[:, 7:27], torch.randn(20, device="cuda")[None].expand(3, 20)):
        assert torch.equal(vig_b200.gated_recurrence(x, x, h0, True)[1], h0)


def test_normalizers_that_no_float_holds_are_refused():
    x = torch.zeros(1, 4, 8, device="cuda")
    for n in (1e-50, 1e-40, 1e40, float("inf")):
        with pytest.raises(ValueError):
            vig_b200.gated_recurrence(x, x, gate_logit_normalizer=n)


@pytest.mark.parametrize("D,reverse", [(1024, False), (1024, True), (1001, False)])
def test_offsets_beyond_32_bits(D, reverse):
    """More than 2^31 values: the far end against a call on its last 3000 tokens alone.  With decays of a sigmoid of normal logits 4000 tokens
    forget what was before them; both calls then round states that agree to 1e-6."""
    L, n = 2_300_000, 3000
    gen = torch.Generator(device="cuda").manual_seed(8)
    x, g = (torch.empty(1, L, D, dtype=torch.bfloat16, device="cuda").normal_(generator=gen) for _ in range(2))
    kw = dict(gate_logit_normalizer=1.0, reverse=reverse)
    h, _ = vig_b200.gated_recurrence(x, g, **kw)
    state = None if reverse else vig_b200.gated_recurrence(x[:, -n - 4000:-n], g[:, -n - 4000:-n], None, True, **kw)[1]
    ref = vig_b200.gated_recurrence(x[:, -n:], g[:, -n:], state, **kw)[0].float()
    assert ((h[:, -n:].float() - ref).abs() <= 2 * UNIT[torch.bfloat16] * ref.abs() + 1e-5).all()
