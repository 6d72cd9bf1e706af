"""The selective scan against its definition in 64 bits, token by token, with all gradients written out.

Tolerances: with u = 2^-24, a decay exp(delta A) is off by at most e = (8 + 24 |delta A|) u of itself (exp2 to 2 ulp, its argument and the step delta, a polynomial, to 16 u), so a product
of up to L of them by L (e + 4 u); that happens in the states and once more in what goes back.  Sums add one u for every term: N states, D channels of a group, B L
tokens.  With G the sum of these, an output is off by at most G times the same sum taken over magnitudes, and by the rounding to its type."""
import math

import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
UNIT = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}
NAMES = ("u", "dt", "A", "B", "C", "D", "z", "dt_bias", "initial_state")


def make(B, L, D, N, G, dtype, seed, z=True, skip=True, bias=True, state=True, param=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    maps = (B, L, N) if G == 0 else (B, L, G, N)
    return dict(u=rand(B, L, D).to(dtype), dt=(0.5 * rand(B, L, D)).to(dtype), A=-torch.rand(D, N, generator=gen) * 4 - 0.05, B=rand(*maps).to(dtype), C=rand(*maps).to(dtype),
                D=rand(D).to(param) if skip else None, z=rand(B, L, D).to(dtype) if z else None, dt_bias=(rand(D) - 2).to(param) if bias else None,
                initial_state=rand(B, D, N) if state else None)


def reference(t, d_y=None, d_final=None, lengths=None, softplus=True):
    """(outputs, their magnitudes): y, final state and, with d_y, the gradients of all inputs, the latter from the same sums over absolute values."""
    w = {k: None if v is None else v.double() for k, v in t.items()}
    Bn, L, D = w["u"].shape
    N = w["A"].shape[1]
    Bm, Cm = (w[k] if w[k].dim() == 4 else w[k][:, :, None] for k in "BC")
    G = Bm.shape[2]
    pick = torch.arange(D) // max(1, D // G)
    inside = torch.ones(Bn, L, 1).double() if lengths is None else (torch.arange(L) < lengths[:, None]).double()[..., None]
    x = w["dt"] + (w["dt_bias"] if w["dt_bias"] is not None else 0)
    delta = torch.where(inside > 0, torch.nn.functional.softplus(x, threshold=60.0) if softplus else x, torch.zeros(()).double())
    keep = lambda v: torch.where(inside > 0, v, torch.zeros(()).double())  # noqa: E731
    u, z = keep(w["u"]), w["z"]
    Bm, Cm = (torch.where(inside[..., None] > 0, m, torch.zeros(()).double()) for m in (Bm, Cm))
    skip = w["D"] if w["D"] is not None else torch.zeros(D).double()
    gate = torch.nn.functional.silu(z) if z is not None else torch.ones(Bn, L, D).double()
    slope = torch.sigmoid(x) if softplus else torch.ones_like(x)
    a = torch.exp(delta[..., None] * w["A"])
    results = []
    for f in (lambda v: v, torch.abs):
        h = f(w["initial_state"]) if w["initial_state"] is not None else torch.zeros(Bn, D, N).double()
        fu, fd, fB, fC, fs, fg, fA = f(u), f(delta), f(Bm), f(Cm), f(skip), f(gate), f(w["A"])
        befores, hs, ys = [], [], torch.zeros(Bn, L, D).double()
        for i in range(L):
            befores.append(h)
            h = a[:, i] * h + (fd[:, i] * fu[:, i])[..., None] * fB[:, i][:, pick]
            hs.append(h)
            ys[:, i] = (h * fC[:, i][:, pick]).sum(-1) + fs * fu[:, i]
        outs = [keep(ys * fg), h]
        if d_y is not None:
            dy, g = f(keep(d_y.double())), f(d_final.double()) if d_final is not None else torch.zeros_like(h)
            dys = dy * fg
            grads = dict(u=torch.zeros_like(u), dt=torch.zeros_like(u), A=torch.zeros_like(w["A"]), B=torch.zeros_like(Bm), C=torch.zeros_like(Bm))
            for i in reversed(range(L)):
                g = g + dys[:, i, :, None] * fC[:, i][:, pick]
                xb = (fd[:, i] * fu[:, i])[..., None]
                grads["C"][:, i].index_add_(1, pick, hs[i] * dys[:, i, :, None])
                grads["B"][:, i].index_add_(1, pick, g * xb)
                along = (g * fB[:, i][:, pick]).sum(-1)
                flow = g * a[:, i] * befores[i]
                grads["A"] += (flow * fd[:, i, :, None]).sum(0)
                grads["dt"][:, i] = ((flow * fA).sum(-1) + along * fu[:, i]) * slope[:, i]
                grads["u"][:, i] = along * fd[:, i] + fs * dys[:, i]
                g = g * a[:, i]
            grads["u"], grads["dt"] = keep(grads["u"]), keep(grads["dt"])
            grads["D"], grads["dt_bias"], grads["initial_state"] = (dys * fu).sum((0, 1)), grads["dt"].sum((0, 1)), g
            if z is not None:
                p = torch.sigmoid(z)
                grads["z"] = dy * ys * f(p * (1 + z * (1 - p)))
            outs += [grads[k].reshape(t[k].shape) if t[k] is not None else None for k in NAMES]
        results.append(outs)
    grow = float((8 + 24 * (delta[..., None] * w["A"]).abs().amax() if delta.numel() else 8) + 4) * U
    room = 2 * L * grow + (64 + 4 * (float(z.abs().max()) if z is not None and z.numel() else 0) + N + D // G + Bn * L) * U
    return results[0], results[1], room


def check(got, ref, mag, room, what=""):
    got = got.double().cpu()
    most = room * mag
    most = most + UNIT[got_type(what)] * (ref.abs() + most) + TINY[got_type(what)]
    off = (got - ref).abs()
    assert torch.isfinite(got).all(), what
    assert (off <= most).all(), f"{what}: worst {float((off / most).max()):.2f} of the bound"


def got_type(what):
    return what[1]


def run(t, lengths=None, d_y=None, d_final=None, softplus=True, want_final=True):
    leaf = {k: None if v is None else v.cuda() for k, v in t.items()}
    if d_y is None:
        with torch.no_grad():
            return vig_b200.selective_scan(**leaf, output_final_state=want_final, dt_softplus=softplus, lengths=lengths)
    leaf = {k: None if v is None else v.requires_grad_(True) for k, v in leaf.items()}
    y, final = vig_b200.selective_scan(**leaf, output_final_state=True, dt_softplus=softplus, lengths=lengths)
    grads = torch.autograd.grad([y, final], [v for v in leaf.values() if v is not None], [d_y.cuda(), d_final.cuda()])
    grads = iter(grads)
    return (y, final, *[None if v is None else next(grads) for v in leaf.values()])


def compare(t, lengths=None, softplus=True, seed=0):
    gen = torch.Generator().manual_seed(seed + 99)
    d_y = torch.randn(t["u"].shape, generator=gen).to(t["u"].dtype)
    d_final = torch.randn(t["u"].shape[0], *t["A"].shape, generator=gen)
    ref, mag, room = reference(t, d_y, d_final, lengths, softplus)
    outs = run(t, None if lengths is None else lengths.cuda(), d_y, d_final, softplus)
    for name, o, r, m in zip(("y", "final", *NAMES), outs, ref, mag):
        if o is None:
            continue
        want = torch.float32 if name in ("final", "A", "initial_state") else t[name].dtype if name in NAMES else t["u"].dtype
        assert o.dtype == want and o.shape == r.shape
        check(o, r, m, room, (name, o.dtype))
    return outs


SHAPES = [(1, 1, 1, 1, 0), (2, 1, 3, 5, 0), (1, 2, 16, 16, 1), (2, 7, 17, 8, 0), (1, 63, 5, 9, 0), (3, 64, 8, 16, 0), (1, 65, 40, 16, 4), (2, 129, 34, 17, 2), (1, 200, 6, 40, 0), (1, 300, 4, 64, 0),
          (2, 130, 20, 2, 0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,L,D,N,G", SHAPES)
def test_forward_and_gradients(B, L, D, N, G, dtype):
    k = SHAPES.index((B, L, D, N, G))
    t = make(B, L, D, N, G, dtype, seed=k, z=k % 3 != 1, skip=k % 4 != 2, bias=k % 5 != 3, state=k % 2 == 0, param=torch.float32 if k % 2 else dtype)
    if k % 6 == 4:
        t["dt"].abs_()          # without softplus a negative step is a state that grows without bound
        t["dt_bias"] = None if t["dt_bias"] is None else t["dt_bias"].abs()
    compare(t, softplus=k % 6 != 4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths", [[0, 1, 70, 64], [130, 129, 65, 2]])
def test_lengths(dtype, lengths):
    """Behind a sequence's end neither inputs nor gradients count, whatever stands there; the outputs there are zeros and the state is the one at the end."""
    t = make(4, 130, 18, 16, 0, dtype, seed=5)
    n = torch.tensor(lengths, dtype=torch.int32)
    clean = compare(t, n)
    behind = torch.arange(130) >= n[:, None]
    for k, bad in (("u", float("nan")), ("dt", float("inf")), ("B", float("nan")), ("C", float("-inf")), ("z", float("nan"))):
        t[k] = torch.where(behind[..., None], torch.tensor(bad).to(dtype), t[k])
    gen = torch.Generator().manual_seed(99)
    d_y = torch.randn(t["u"].shape, generator=gen).to(dtype)
    d_final = torch.randn(4, 18, 16, generator=gen)
    dirty = run(t, n.long().cuda(), torch.where(behind[..., None], torch.tensor(float("nan")).to(dtype), d_y), d_final)
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)
    assert not clean[0][behind.cuda()].any()
    out_of_range = run({k: v for k, v in make(4, 130, 18, 16, 0, dtype, seed=5).items()}, torch.tensor([-3, 1 << 30, 131, 130], dtype=torch.int32).cuda())[0]
    whole = run(make(4, 130, 18, 16, 0, dtype, seed=5), torch.tensor([0, 130, 130, 130], dtype=torch.int32).cuda())[0]
    assert torch.equal(out_of_range, whole)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,D,N", [(1, 1500, 768, 16), (20, 200, 256, 16), (12, 130, 512, 8), (40, 70, 128, 16), (40, 128, 256, 16), (80, 60, 256, 16), (90, 100, 256, 5)])
def test_every_width_of_a_block(B, L, D, N, dtype):
    """Few, some and many channels: sequences of a larger call against calls of their own, and against 64 bits."""
    t = make(B, L, D, N, 0, dtype, seed=3)
    y, final = run(t)
    b = B - 1
    one = {k: v if k in ("A", "D", "dt_bias") else v[b:b + 1] for k, v in t.items()}
    some = {k: v[:24] if k in ("A", "D", "dt_bias") else v[..., :24] if k in ("u", "dt", "z") else v[:, :24] if k == "initial_state" else v for k, v in one.items()}
    ref, mag, room = reference(some)
    check(y[b:b + 1, :, :24], ref[0], mag[0], room, ("y", dtype))
    check(final[b:b + 1, :24], ref[1], mag[1], room, ("final", torch.float32))


def test_runs_joined_give_the_whole():
    """A prefix read in, then the rest from its state: the same bits as the tiles of 64 are the same."""
    t = make(2, 256, 40, 16, 0, torch.bfloat16, seed=9)
    y, final = run(t)
    first = {k: v[:, :128] if k in ("u", "dt", "B", "C", "z") else v for k, v in t.items()}
    y1, s1 = run(first)
    rest = {k: v[:, 128:] if k in ("u", "dt", "B", "C", "z") else v for k, v in t.items()}
    rest["initial_state"] = s1.cpu()
    y2, s2 = run(rest)
    assert torch.equal(torch.cat([y1, y2], 1), y) and torch.equal(s2, final)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,D,N,G", [(1, 1, 1, 0), (3, 7, 5, 0), (8, 768, 16, 0), (2, 66, 64, 2), (5, 33, 17, 3)])
def test_step(B, D, N, G, dtype):
    t = make(B, 1, D, N, G, dtype, seed=N, z=D != 7, skip=D != 33, bias=D != 66, param=dtype if D == 7 else torch.float32)
    ref, mag, room = reference(t)
    table = torch.full((B, 3, D, N), float("nan"), device="cuda")
    state = table[:, 1]
    state.copy_(t["initial_state"])
    at = lambda k: None if t[k] is None else t[k][:, 0].cuda()  # noqa: E731
    before = state._version
    y = vig_b200.selective_scan_step(at("u"), at("dt"), t["A"].cuda(), at("B"), at("C"), state, None if t["D"] is None else t["D"].cuda(), at("z"),
                                     None if t["dt_bias"] is None else t["dt_bias"].cuda())
    check(y, ref[0][:, 0], mag[0][:, 0], room, ("y", dtype))
    check(state, ref[1], mag[1], room, ("state", torch.float32))
    assert state._version > before and table[:, 0].isnan().all() and table[:, 2].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views(dtype):
    """Slices of wider projections, rows that begin anywhere, maps without room between and one map for all sequences, states of a larger table."""
    t = make(2, 70, 24, 10, 0, dtype, seed=1)
    plain = run(t)
    g = {k: None if v is None else v.cuda() for k, v in t.items()}
    wide = torch.randn(2, 70, 3 * 24 + 2 * 10 + 1, device="cuda").to(dtype)
    cuts = dict(u=(1, 25), dt=(25, 49), z=(49, 73), B=(73, 83), C=(83, 93))
    for k, (i, j) in cuts.items():
        wide[..., i:j] = g[k]
        g[k] = wide[..., i:j]
    table = torch.zeros(2, 2, 24, 10, device="cuda")
    table[:, 1] = g["initial_state"]
    g["initial_state"] = table[:, 1]
    with torch.no_grad():
        y, final = vig_b200.selective_scan(**g, output_final_state=True)
    assert torch.equal(y, plain[0]) and torch.equal(final, plain[1])
    with torch.no_grad():
        same = vig_b200.selective_scan(g["u"], g["dt"], g["A"], g["B"][:1].expand(2, -1, -1), g["C"][:1].expand(2, -1, -1))[0]
        each = vig_b200.selective_scan(g["u"], g["dt"], g["A"], g["B"][:1].repeat(2, 1, 1), g["C"][:1].repeat(2, 1, 1))[0]
    assert torch.equal(same, each)


def test_empty_calls():
    for B, L, D in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        t = make(B, L, D, 4, 0, torch.float32, seed=0)
        d_f = torch.randn(B, D, 4)
        outs = run(t, None, torch.zeros(B, L, D), d_f)
        assert outs[0].shape == (B, L, D) and outs[1].shape == (B, D, 4)
        if L == 0:
            assert torch.equal(outs[1].cpu(), t["initial_state"]) and torch.equal(outs[-1].cpu(), d_f)
        for k, g in zip(NAMES, outs[2:]):
            assert g.shape == t[k].shape and (k == "initial_state" or not g.any())


def test_infinities_stay():
    """A state that is infinite stays so over products of decays that have left fp32's range, within a tile and from tile to tile."""
    t = make(1, 400, 16, 16, 0, torch.float32, seed=2, skip=False, z=False, bias=False)
    t["dt"].fill_(2.0)
    t["initial_state"][0, 3, 5] = float("inf")
    t["initial_state"][0, 4, 1] = float("-inf")
    t["A"][:5] = -1.0
    final = run(t)[1].cpu()
    assert final[0, 3, 5] == float("inf") and final[0, 4, 1] == float("-inf")
    final[0, 3, 5] = final[0, 4, 1] = 0
    assert torch.isfinite(final).all()
    t["B"][0, 70, 2] = float("inf")
    t["u"].abs_()
    final = run(t)[1].cpu()
    assert (final[0, :, 2] == float("inf")).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_steps_of_nothing(dtype):
    """A raw step of -inf, or of the type's lowest value, is one of nothing: the state passes as it was, the token has no gradient but the skip's, and nothing becomes a NaN."""
    t = make(2, 100, 20, 16, 0, dtype, seed=7)
    for i, v in enumerate((float("-inf"), torch.finfo(dtype).min)):
        t["dt"][i, 10:80] = v
    outs = compare(t)
    assert not outs[3][:, 10:80].any()                           # the gradient of dt
    c = {k: v.cuda() for k, v in t.items()}
    state = c["initial_state"].clone()
    y = vig_b200.selective_scan_step(c["u"][:, 20], c["dt"][:, 20], c["A"], c["B"][:, 20], c["C"][:, 20], state, c["D"], c["z"][:, 20], c["dt_bias"])
    assert torch.equal(state, c["initial_state"]) and torch.isfinite(y).all()
    t["dt"][0, 50, 3] = float("nan")
    y, final = run(t)
    assert y[0, 50:, 3].isnan().all() and final[0, 3].isnan().all()
    y[0, :, 3] = final[0, 3] = 0
    assert torch.isfinite(y).all() and torch.isfinite(final).all()
    t["dt"][0, 50, 3], t["dt"][1, 60, 4], t["u"][1, 60, 4] = 0, float("inf"), 1
    y, final = run(t)
    assert not torch.isfinite(final[1, 4]).any() and torch.isfinite(final[0]).all()


def test_graph_and_streams():
    """Captured with its backward and replayed on other values; on a stream of its own; the same bits every time."""
    t = make(2, 150, 48, 16, 0, torch.bfloat16, seed=4)
    d_y, d_f = torch.randn(2, 150, 48).bfloat16(), torch.randn(2, 48, 16)
    eager = run(t, None, d_y, d_f)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        other = run(t, None, d_y, d_f)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    leaf = {k: torch.zeros_like(v, device="cuda").requires_grad_(True) for k, v in t.items()}
    gy, gf = torch.zeros_like(d_y, device="cuda"), torch.zeros_like(d_f, device="cuda")

    def step():
        y, f = vig_b200.selective_scan(**leaf, output_final_state=True)
        return (y, f, *torch.autograd.grad([y, f], list(leaf.values()), [gy, gf]))

    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = step()
    with torch.no_grad():
        for k, v in leaf.items():
            v.copy_(t[k])
    gy.copy_(d_y)
    gf.copy_(d_f)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, outs))


def test_gradients_against_differences():
    t = {k: v.double() if v is not None else v for k, v in make(1, 20, 3, 4, 0, torch.float32, seed=6).items()}
    gen = torch.Generator().manual_seed(0)
    d_y, d_f = torch.randn(1, 20, 3, generator=gen), torch.randn(1, 3, 4, generator=gen)
    grads = run({k: v.float() for k, v in t.items()}, None, d_y, d_f)[2:]
    loss = lambda w: float((reference(w)[0][0] * d_y).sum() + (reference(w)[0][1] * d_f).sum())  # noqa: E731
    for k, g in zip(NAMES, grads):
        at = tuple(torch.randint(0, n, (), generator=gen).item() for n in t[k].shape)
        moved = {**t, k: t[k].clone()}
        moved[k][at] += 1e-5
        up = loss(moved)
        moved[k][at] -= 2e-5
        diff = (up - loss(moved)) / 2e-5
        assert abs(float(g[at]) - diff) <= 1e-4 * (1 + abs(diff)), k


def test_far_rows():
    """Sequences more than 2^31 elements apart."""
    t = make(2, 66, 16, 16, 0, torch.bfloat16, seed=8, state=False)
    plain = run(t)
    far = torch.empty(2 ** 31 + 66 * 16 + 64, dtype=torch.bfloat16, device="cuda")
    g = {k: None if v is None else v.cuda() for k, v in t.items()}
    u = far.as_strided((2, 66, 16), (2 ** 31, 16, 1))
    u.copy_(g["u"])
    with torch.no_grad():
        y, final = vig_b200.selective_scan(**{**g, "u": u}, output_final_state=True)
    assert torch.equal(y, plain[0]) and torch.equal(final, plain[1])
    del u
    B = far.as_strided((2, 66, 16), (2 ** 31, 16, 1))
    B.copy_(g["B"])
    with torch.no_grad():
        y, final = vig_b200.selective_scan(**{**g, "B": B}, output_final_state=True)
    assert torch.equal(y, plain[0]) and torch.equal(final, plain[1])


def test_refusals():
    t = {k: v.cuda() for k, v in make(2, 8, 6, 4, 0, torch.float32, seed=0).items()}
    call = lambda **kw: vig_b200.selective_scan(**{**t, **kw})  # noqa: E731
    for bad in (dict(dt=t["dt"][:, :7]), dict(u=t["u"].transpose(1, 2)), dict(A=t["A"][:, :3]), dict(A=t["A"].t().contiguous().t()), dict(B=t["B"][..., :3]), dict(C=t["C"][:1]),
                dict(B=t["B"][:, :, None].expand(-1, -1, 4, -1), C=t["C"][:, :, None].expand(-1, -1, 4, -1)), dict(D=t["D"][:5]), dict(initial_state=t["initial_state"][:, :5]),
                dict(initial_state=t["initial_state"].transpose(1, 2)), dict(lengths=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(A=torch.zeros(6, 65, device="cuda"))):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(dt=t["dt"].bfloat16()), dict(A=t["A"].double()), dict(B=t["B"].half()), dict(D=t["D"].half()), dict(u=t["u"].double(), dt=t["dt"].double()),
                dict(lengths=torch.zeros(2, device="cuda")), dict(initial_state=t["initial_state"].half())):
        with pytest.raises(TypeError):
            call(**bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        call(dt=t["dt"].cpu())
    one = lambda k: t[k][:, 0].contiguous()  # noqa: E731
    state = t["initial_state"].clone()
    step = lambda state, **kw: vig_b200.selective_scan_step(kw.get("u", one("u")), one("dt"), t["A"], one("B"), one("C"), state)  # noqa: E731
    for bad in (state[:, :5], state[:1].expand(2, -1, -1), state.transpose(1, 2)):
        with pytest.raises(ValueError):
            step(bad)
    with pytest.raises(NotImplementedError):
        step(state, u=one("u").requires_grad_(True))
    y, _ = vig_b200.selective_scan(**{**t, "u": t["u"].clone().requires_grad_(True)})
    g, = torch.autograd.grad(y.sum(), [y], create_graph=True)
    u = t["u"].clone().requires_grad_(True)
    y, _ = vig_b200.selective_scan(**{**t, "u": u})
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(y.sum(), u, create_graph=True)


def test_step_is_the_scan():
    """Token by token through `selective_scan_step` gives the states that `selective_scan` gives, to the bound of both."""
    t = make(2, 90, 20, 16, 0, torch.float32, seed=12)
    ref, mag, room = reference(t)
    state = t["initial_state"].cuda()
    c = {k: v.cuda() for k, v in t.items()}
    ys = [vig_b200.selective_scan_step(c["u"][:, i], c["dt"][:, i], c["A"], c["B"][:, i], c["C"][:, i], state, c["D"], c["z"][:, i], c["dt_bias"]) for i in range(90)]
    check(torch.stack(ys, 1), ref[0], mag[0], room, ("y", torch.float32))
    check(state, ref[1], mag[1], room, ("state", torch.float32))
    assert math.isfinite(room)
