"""The trainable layer norm against its definition in 64 bits.

Tolerances: with u = 2^-24 and rows of N values, mean and variance come out of sums in any order, off by at most (N + 2) u of the sum of magnitudes; with m = max |r| over a row
and rstd its 1 / deviation, xh is off by e = 2 (N + 8) u (1 + m rstd) at most, and so are the other terms of the gradient beside their own sums."""
import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
UNIT = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
EPS = 1e-5


def make(M, N, dtype, seed, residual=True, bias=True, param=None, mean=0.5):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return dict(x=(rand(M, N) + mean).to(dtype), weight=(1 + 0.2 * rand(N)).to(param or dtype), bias=rand(N).to(param or dtype) if bias else None,
                residual=(2 * rand(M, N)).to(dtype) if residual else None), rand(M, N).to(dtype), rand(M, N).to(dtype)


def reference(t, d_y, d_r):
    r = t["x"].double() + (t["residual"].double() if t["residual"] is not None else 0)
    N = r.shape[-1]
    w, b = t["weight"].double(), t["bias"].double() if t["bias"] is not None else torch.zeros(N).double()
    rstd = 1 / (r.var(-1, keepdim=True, correction=0) + EPS).sqrt()
    xh = (r - r.mean(-1, keepdim=True)) * rstd
    e = 2 * (N + 8) * U * (1 + r.abs().amax(-1, keepdim=True) * rstd)
    y = xh * w + b
    e_y = (e + U * xh.abs()) * w.abs() + 3 * U * (y.abs() + b.abs())
    g = d_y.double()
    s = g * w
    mean_s, dot = s.mean(-1, keepdim=True), (s * xh).mean(-1, keepdim=True)
    dx = rstd * (s - mean_s - xh * dot) + d_r.double()
    mags = s.abs() + s.abs().mean(-1, keepdim=True) + xh.abs() * (s * xh).abs().mean(-1, keepdim=True)
    e_dx = rstd * (mags * ((N + 16) * U + 2 * e) + e * (s.abs().mean(-1, keepdim=True) * (1 + xh.abs()))) + 4 * U * (dx.abs() + d_r.double().abs())
    if t["residual"] is None:
        # r is x itself, so d_r comes to x's gradient by autograd's own addition behind the kernel's: the norm's share, dx - d_r, is rounded to the type once more
        e_dx = e_dx + UNIT[t["x"].dtype] * ((dx - d_r.double()).abs() + e_dx)
    M = r.shape[0]
    dw, e_w = (g * xh).sum(0), (g.abs() * e).sum(0) + (M + 2) * U * (g * xh).abs().sum(0)
    return [(y, e_y), (r, U * r.abs()), (dx, e_dx), (dw, e_w), (g.sum(0), (M + 2) * U * g.abs().sum(0)), (dx, e_dx)]


def check(got, want, what):
    ref, bound = want
    most = bound + UNIT[got.dtype] * (ref.abs() + bound) + 2.0 ** -24
    off = (got.double().cpu() - ref).abs()
    assert got.shape == ref.shape and torch.isfinite(got).all(), what
    assert (off <= most).all(), f"{what}: worst {float((off / most).max()):.2f} of the bound"


def run(t, d_y, d_r):
    leaf = {k: None if v is None else v.requires_grad_(True) for k, v in t.items()}
    y, r = vig_b200.add_layernorm_train(**leaf, eps=EPS)
    grads = iter(torch.autograd.grad([y, r], [v for v in leaf.values() if v is not None], [d_y, d_r]))
    return [y, r] + [None if v is None else next(grads) for v in leaf.values()]


WIDTHS = [1, 2, 7, 8, 31, 33, 96, 100, 192, 333, 384, 768, 1000, 2049, 4096, 9001]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N", WIDTHS)
def test_forward_and_gradients(N, dtype):
    i = WIDTHS.index(N)
    t, d_y, d_r = make(1 + 37 * (i % 4), N, dtype, seed=i, residual=i % 3 != 0, bias=i % 4 != 1, param=torch.float32 if i % 2 else None)
    outs = run({k: None if v is None else v.cuda() for k, v in t.items()}, d_y.cuda(), d_r.cuda())
    refs = reference(t, d_y, d_r)
    for what, o, want in zip(("y", "r", "dx", "dw", "db", "dres"), outs, refs):
        if o is not None:
            check(o, want, what)
    with torch.no_grad():
        g = {k: None if v is None else v.cuda() for k, v in t.items()}
        y, r = vig_b200.add_layernorm_train(**g, eps=EPS)
        dx, dw, db = vig_b200.add_layernorm_backward(d_y.cuda(), g["x"], g["weight"], EPS, d_r.cuda(), g["residual"])
    assert torch.equal(y, outs[0]) and torch.equal(dw, outs[3]) and (t["bias"] is None or torch.equal(db, outs[4]))
    check(dx, refs[2], "dx of the function")


def test_wide_rows():
    """Rows past what a block's threads hold."""
    for dtype, N in ((torch.bfloat16, 16392), (torch.float32, 8200)):
        t, d_y, d_r = make(3, N, dtype, seed=1)
        for what, o, want in zip(("y", "r", "dx", "dw", "db", "dres"), run({k: v.cuda() for k, v in t.items()}, d_y.cuda(), d_r.cuda()), reference(t, d_y, d_r)):
            check(o, want, what)


def test_large_mean():
    """A deviation that is small beside the mean: the variance is that of the differences."""
    t, d_y, d_r = make(5, 384, torch.float32, seed=2, residual=False, mean=1000.0)
    for what, o, want in zip(("y", "r", "dx", "dw", "db"), run({k: None if v is None else v.cuda() for k, v in t.items()}, d_y.cuda(), d_r.cuda()), reference(t, d_y, d_r)):
        check(o, want, what)
    y = run({k: None if v is None else v.cuda() for k, v in t.items()}, d_y.cuda(), d_r.cuda())[0]
    plain = torch.nn.functional.layer_norm(t["x"].double(), (384,), t["weight"].double(), t["bias"].double(), EPS)
    assert float((y.double().cpu() - plain).abs().max()) < 1e-2


def test_rows_of_equal_values():
    x = torch.full((4, 96), 3.0, device="cuda").requires_grad_(True)
    w = torch.ones(96, device="cuda").requires_grad_(True)
    y, _ = vig_b200.add_layernorm_train(x, w)
    dx, dw = torch.autograd.grad(y.sum(), [x, w])
    assert not y.any() and not dw.any() and torch.isfinite(dx).all()


def test_views_shapes_and_graph():
    t, d_y, d_r = make(60, 96, torch.bfloat16, seed=4)
    g = {k: v.cuda() for k, v in t.items()}
    plain = run(dict(g), d_y.cuda(), d_r.cuda())
    wide = torch.zeros(60, 96 + 40, device="cuda", dtype=torch.bfloat16)
    for first in (0, 1, 16):
        wide[:, first:first + 96] = g["x"].detach()
        y, r = vig_b200.add_layernorm_train(wide[:, first:first + 96], g["weight"].detach(), g["bias"].detach(), g["residual"].detach(), EPS)
        assert torch.equal(y, plain[0]) and torch.equal(r, plain[1])
    y, _ = vig_b200.add_layernorm_train(g["x"].detach().view(3, 4, 5, 96), g["weight"].detach(), g["bias"].detach(), g["residual"].detach().view(3, 4, 5, 96), EPS)
    assert y.shape == (3, 4, 5, 96) and torch.equal(y.view(60, 96), plain[0])
    leaf = {k: torch.zeros_like(v).requires_grad_(True) for k, v in g.items()}
    gy, gr = d_y.cuda(), d_r.cuda()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        run(dict(leaf), gy, gr)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = run(dict(leaf), gy, gr)
    with torch.no_grad():
        for k, v in leaf.items():
            v.copy_(g[k])
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(plain, outs))


def test_empty_and_refusals():
    x, w = torch.zeros(0, 8, device="cuda", requires_grad=True), torch.ones(8, device="cuda", requires_grad=True)
    y, r = vig_b200.add_layernorm_train(x, w, w)
    dw, = torch.autograd.grad(y.sum(), [w])
    assert y.shape == (0, 8) and not dw.any()
    x, w = torch.zeros(4, 8, device="cuda"), torch.ones(8, device="cuda")
    for bad in (dict(weight=w[:7]), dict(bias=w[:7]), dict(residual=x[:3]), dict(eps=-1.0), dict(x=torch.zeros(4, 0, device="cuda"), weight=torch.zeros(0, device="cuda"))):
        with pytest.raises(ValueError):
            vig_b200.add_layernorm_train(**{**dict(x=x, weight=w), **bad})
    for bad in (dict(x=x.double()), dict(weight=w.half()), dict(bias=w.half()), dict(residual=x.half())):
        with pytest.raises(TypeError):
            vig_b200.add_layernorm_train(**{**dict(x=x, weight=w), **bad})
