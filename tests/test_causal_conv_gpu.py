"""The short causal convolution against its definition in 64 bits, tap by tap, with all gradients written out.

Tolerances: with u = 2^-24 a sum of n terms is off by at most (n + 1) u of the sum of their magnitudes; silu and its slope, from exp2 and a reciprocal, by (16 + 4 |pre|) u of
themselves, and by their slope, at most 1.1, times the error of pre.  Then the rounding to the output's type."""
import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
UNIT = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}


def make(B, L, D, K, dtype, seed, bias=True, state=True, param=None):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return dict(x=rand(B, L, D).to(dtype), weight=rand(D, K).to(param or dtype), bias=rand(D).to(param or dtype) if bias else None,
                initial_state=rand(B, K - 1, D).to(dtype) if state else None)


def reference(t, silu, d_y=None, d_final=None, lengths=None):
    """[(value, bound of its error before rounding)]: y, final state, gradients of x, weight, bias, initial_state"""
    x, w = t["x"].double(), t["weight"].double()
    B, L, D = x.shape
    K = w.shape[1]
    ends = [L] * B if lengths is None else lengths.tolist()
    inside = torch.tensor([[i < e for i in range(L)] for e in ends]).view(B, L, 1)
    x = torch.where(inside, x, torch.zeros(()).double())
    front = t["initial_state"].double() if t["initial_state"] is not None else torch.zeros(B, K - 1, D).double()
    whole = torch.cat([front, x], 1)
    bias = t["bias"].double() if t["bias"] is not None else torch.zeros(D).double()
    pre, mag = bias.expand(B, L, D).clone(), bias.abs().expand(B, L, D).clone()
    for k in range(K):
        pre += w[:, k] * whole[:, k:k + L]
        mag += (w[:, k] * whole[:, k:k + L]).abs()
    e_pre = (K + 2) * U * mag
    s = torch.sigmoid(pre)
    rel = (16 + 4 * pre.abs()) * U
    y, e_y = (pre * s, 1.1 * e_pre + rel * (pre * s).abs()) if silu else (pre, e_pre)
    zero = torch.zeros(()).double()
    outs = [(torch.where(inside, y, zero), e_y), (torch.stack([whole[b, e:e + K - 1] for b, e in enumerate(ends)]), torch.zeros(()).double())]
    if d_y is None:
        return outs
    dy = torch.where(inside, d_y.double(), zero)
    slope = s * (1 + pre * (1 - s)) if silu else torch.ones_like(pre)
    g = dy * slope
    e_g = dy.abs() * (0.6 * e_pre + rel * (s * (1 + pre.abs()))) + U * g.abs() if silu else torch.zeros_like(g)   # |silu''| <= 0.5
    d_whole, e_whole, m_whole = (torch.zeros_like(whole) for _ in range(3))
    dw, e_w, m_w = (torch.zeros(D, K).double() for _ in range(3))
    for k in range(K):
        d_whole[:, k:k + L] += w[:, k] * g
        m_whole[:, k:k + L] += (w[:, k] * g).abs()
        e_whole[:, k:k + L] += w[:, k].abs() * e_g
        dw[:, k] = (g * whole[:, k:k + L]).sum((0, 1))
        m_w[:, k] = (g * whole[:, k:k + L]).abs().sum((0, 1))
        e_w[:, k] = (e_g * whole[:, k:k + L].abs()).sum((0, 1))
    for b, e in enumerate(ends):
        d_whole[b, e:e + K - 1] += d_final[b].double()
        m_whole[b, e:e + K - 1] += d_final[b].double().abs()
    e_whole = e_whole + (K + 3) * U * m_whole
    n = (B * L + 2) * U
    outs += [(torch.where(inside, d_whole[:, K - 1:], zero), e_whole[:, K - 1:]), (dw, e_w + n * m_w), (g.sum((0, 1)), e_g.sum((0, 1)) + n * g.abs().sum((0, 1))),
             (d_whole[:, :K - 1], e_whole[:, :K - 1])]
    return outs


def check(got, want, what):
    ref, bound = want
    most = bound + UNIT[got.dtype] * (ref.abs() + bound) + TINY[got.dtype]
    off = (got.double().cpu() - ref).abs()
    assert got.shape == ref.shape and torch.isfinite(got).all(), what
    assert (off <= most).all(), f"{what}: worst {float((off / most).max()):.2f} of the bound"


def compare(t, silu, lengths=None):
    B, L, D = t["x"].shape
    K = t["weight"].shape[1]
    gen = torch.Generator().manual_seed(1)
    d_y, d_f = torch.randn(B, L, D, generator=gen).to(t["x"].dtype), torch.randn(B, K - 1, D, generator=gen).to(t["x"].dtype)
    leaf = {k: None if v is None else v.cuda().requires_grad_(True) for k, v in t.items()}
    y, final = vig_b200.causal_conv(**leaf, output_final_state=True, activation="silu" if silu else None, lengths=None if lengths is None else lengths.cuda())
    grads = iter(torch.autograd.grad([y, final], [v for v in leaf.values() if v is not None], [d_y.cuda(), d_f.cuda()]))
    outs = [y, final] + [None if v is None else next(grads) for v in leaf.values()]
    for what, o, want in zip(("y", "final", *t), outs, reference(t, silu, d_y, d_f, lengths)):
        if o is not None:
            check(o, want, what)
    with torch.no_grad():
        again, f2 = vig_b200.causal_conv(**{k: None if v is None else v.detach() for k, v in leaf.items()}, output_final_state=True, activation="silu" if silu else None,
                                         lengths=None if lengths is None else lengths.cuda())
    assert torch.equal(again, y) and torch.equal(f2, final)
    return outs


SHAPES = [(1, 1, 1), (2, 1, 8), (1, 2, 5), (3, 3, 7), (2, 9, 64), (1, 33, 130), (2, 65, 36), (1, 200, 4), (5, 40, 257), (1, 700, 128)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("B,L,D", SHAPES)
def test_forward_and_gradients(B, L, D, K, dtype):
    i = SHAPES.index((B, L, D)) + K
    compare(make(B, L, D, K, dtype, seed=i, bias=i % 3 != 0, state=i % 2 == 0, param=torch.float32 if i % 4 == 1 else None), silu=i % 5 != 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [2, 4])
def test_lengths(K, dtype):
    t = make(6, 40, 12, K, dtype, seed=3)
    n = torch.tensor([0, 1, 2, 39, 40, 17], dtype=torch.int32)
    clean = compare(t, True, n)
    behind = (torch.arange(40) >= n[:, None])[..., None]
    dirty = dict(t, x=torch.where(behind, torch.tensor(float("nan")).to(dtype), t["x"]))
    gen = torch.Generator().manual_seed(1)
    d_y, d_f = torch.randn(6, 40, 12, generator=gen).to(dtype), torch.randn(6, K - 1, 12, generator=gen).to(dtype)
    leaf = {k: v.cuda().requires_grad_(True) for k, v in dirty.items()}
    y, final = vig_b200.causal_conv(**leaf, output_final_state=True, activation="silu", lengths=n.long().cuda())
    grads = torch.autograd.grad([y, final], list(leaf.values()), [torch.where(behind, torch.tensor(float("nan")).to(dtype), d_y).cuda(), d_f.cuda()])
    for a, b in zip(clean, (y, final, *grads)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,D,K", [(1, 1, 1), (3, 7, 3), (8, 768, 4), (2, 130, 8)])
def test_step(B, D, K, dtype):
    """Token by token: the outputs and windows of the whole, bit for bit; windows may lie with the taps outside."""
    t = {k: None if v is None else v.cuda() for k, v in make(B, 12, D, K, dtype, seed=K).items()}
    with torch.no_grad():
        y, final = vig_b200.causal_conv(**t, output_final_state=True, activation="silu")
    table = torch.zeros(K - 1, B, D, dtype=dtype, device="cuda")
    state = table.transpose(0, 1)
    state.copy_(t["initial_state"])
    ys = [vig_b200.causal_conv_step(t["x"][:, i], state, t["weight"], t["bias"], activation="silu") for i in range(12)]
    assert torch.equal(state, final)
    torch.testing.assert_close(torch.stack(ys, 1).double(), y.double(), rtol=2 * UNIT[dtype] + 32 * U, atol=(K + 2) * 16 * U)


def test_views_and_streams():
    t = make(2, 50, 16, 4, torch.bfloat16, seed=2)
    g = {k: v.cuda() for k, v in t.items()}
    with torch.no_grad():
        plain = vig_b200.causal_conv(**g, output_final_state=True)
        for first in (0, 1, 8):
            wide = torch.randn(2, 50, 41, device="cuda").bfloat16()
            wide[..., first:first + 16] = g["x"]
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                y, final = vig_b200.causal_conv(**{**g, "x": wide[..., first:first + 16]}, output_final_state=True)
            stream.synchronize()
            assert torch.equal(y, plain[0]) and torch.equal(final, plain[1])
        far = torch.empty(2 ** 31 + 50 * 16, dtype=torch.bfloat16, device="cuda").as_strided((2, 50, 16), (2 ** 31, 16, 1))
        far.copy_(g["x"])
        y, final = vig_b200.causal_conv(**{**g, "x": far}, output_final_state=True)
        assert torch.equal(y, plain[0]) and torch.equal(final, plain[1])


def test_graph():
    t = make(3, 70, 24, 4, torch.bfloat16, seed=2)
    eager = compare(t, True)
    leaf = {k: torch.zeros_like(v, device="cuda").requires_grad_(True) for k, v in t.items()}
    gen = torch.Generator().manual_seed(1)
    d_y, d_f = torch.randn(3, 70, 24, generator=gen).bfloat16().cuda(), torch.randn(3, 3, 24, generator=gen).bfloat16().cuda()

    def step():
        y, f = vig_b200.causal_conv(**leaf, output_final_state=True, activation="silu")
        return (y, f, *torch.autograd.grad([y, f], list(leaf.values()), [d_y, d_f]))

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = step()
    with torch.no_grad():
        for k, v in leaf.items():
            v.copy_(t[k])
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, outs))


def test_empty_and_refusals():
    for B, L, D in ((0, 4, 8), (2, 0, 8), (2, 4, 0)):
        t = make(B, L, D, 4, torch.float32, seed=0)
        leaf = {k: v.cuda().requires_grad_(True) for k, v in t.items()}
        y, final = vig_b200.causal_conv(**leaf, output_final_state=True)
        assert y.shape == (B, L, D) and final.shape == (B, 3, D)
        if L == 0:
            assert torch.equal(final, leaf["initial_state"])
        grads = torch.autograd.grad([y, final], list(leaf.values()), [torch.ones_like(y), torch.ones_like(final)])
        assert not grads[0].any() and not grads[1].any() and not grads[2].any() and (grads[3] == (1 if L == 0 else grads[3])).all()
    t = {k: v.cuda() for k, v in make(2, 8, 6, 4, torch.float32, seed=0).items()}
    call = lambda **kw: vig_b200.causal_conv(**{**t, **kw})  # noqa: E731
    for bad in (dict(x=t["x"].transpose(1, 2)), dict(x=t["x"][0]), dict(weight=t["weight"][:5]), dict(weight=torch.zeros(6, 9, device="cuda")), dict(weight=t["weight"].t().contiguous().t()),
                dict(bias=t["bias"][:5]), dict(initial_state=t["initial_state"][:, :2]), dict(lengths=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(activation="relu")):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(x=t["x"].double()), dict(weight=t["weight"].half(), bias=None), dict(bias=t["bias"].half()), dict(initial_state=t["initial_state"].half())):
        with pytest.raises(TypeError):
            call(**bad)
    state, x = t["initial_state"], t["x"][:, 0]
    for bad in (state[:1].expand(2, -1, -1), state[:, :1].expand(-1, 3, -1), state[:, :2]):
        with pytest.raises(ValueError):
            vig_b200.causal_conv_step(x, bad, t["weight"])
    with pytest.raises(NotImplementedError):
        vig_b200.causal_conv_step(x, state, t["weight"].clone().requires_grad_(True))
