"""RMS norm with 8-bit rows and its training form against the formulas in 64 bits.

Tolerances: with u = 2^-24 a sum of N squares is off by at most (N/W + log2 W + 2) u of itself for W partial sums (W >= 8 here), so rstd
by half of that and 4 u for its root and reciprocal, y by another 3 u, a scale by 2 u more.  A code stands for a value within half a step
of its type (e4m3: 1/16 of the value, or 2^-10 where codes are subnormal; int8: 1/2), plus what y and the scale are off."""
import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
UNIT = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-6


def rel_rstd(N):
    return (N / 8 + 8) * U / 2 + 4 * U


def make(M, N, dtype, seed, residual, w_dtype=None):
    gen = torch.Generator().manual_seed(seed)
    x, res = torch.randn(M, N, generator=gen).to(dtype), (2 * torch.randn(M, N, generator=gen)).to(dtype) if residual else None
    return x, (1 + 0.3 * torch.randn(N, generator=gen)).to(w_dtype or dtype), res


def formula(x, w, res):
    r = x.double() + (res.double() if res is not None else 0)
    rstd = (r.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return r, rstd, r * rstd * w.double()


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def check8(q, scale, y, group, out):
    N = y.shape[-1]
    width = group or N
    rel = rel_rstd(N) + 8 * U
    rows = y.unflatten(-1, (-1, width))
    want = rows.abs().amax(-1) / (448 if out == torch.float8_e4m3fn else 127)
    scale = scale.cpu().double()
    assert scale.shape == want.shape
    assert ((scale - want).abs() <= rel * want).all()
    stood = q.cpu().to(torch.float64).unflatten(-1, (-1, width)) * scale[..., None]
    unit = scale[..., None]
    half = torch.maximum(rows.abs() / 16, unit * 2.0 ** -10) if out == torch.float8_e4m3fn else unit / 2
    assert ((stood - rows).abs() <= half * (1 + 2.0 ** -10) + 4 * rel * rows.abs()).all()


WIDTHS = [1, 3, 31, 64, 96, 100, 192, 193, 200, 256, 320, 384, 520, 768, 1000, 1024, 1536, 2048, 2056, 4096, 5000, 8192, 9000, 20000]


@pytest.mark.parametrize("out", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", WIDTHS)
def test_rows_in_8_bits(N, dtype, out):
    for M, residual in ((1, True), (5, False), (67, True)):
        x, w, res = make(M, N, dtype, seed=N + M, residual=residual, w_dtype=torch.float32 if M == 5 else None)
        q, scale, r = vig_b200.add_rmsnorm_8bit(*cuda(x, w, res), eps=EPS, dtype=out, prenorm=True)
        rd, _, y = formula(x, w, res)
        assert q.dtype == out and q.shape == x.shape and r.dtype == dtype
        check8(q, scale, y, 0, out)
        assert ((r.cpu().double() - rd).abs() <= UNIT[dtype] * rd.abs() * (1 + 2.0 ** -8) + U * rd.abs() + TINY[dtype]).all()
        again = vig_b200.add_rmsnorm_8bit(*cuda(x, w, res), eps=EPS, dtype=out)
        assert len(again) == 2 and torch.equal(again[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(again[1], scale)


@pytest.mark.parametrize("out", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,group", [(32, 32), (96, 32), (192, 64), (384, 128), (768, 128), (1024, 64), (2048, 32), (128, 128), (640, 128), (4096, 128), (10240, 64), (448, 64)])
def test_groups(N, group, dtype, out):
    for M in (1, 33):
        x, w, res = make(M, N, dtype, seed=N + group, residual=True)
        q, scale = vig_b200.add_rmsnorm_8bit(*cuda(x, w, res), eps=EPS, dtype=out, group=group)
        check8(q, scale, formula(x, w, res)[2], group, out)


@pytest.mark.parametrize("N", [192, 193, 1024])
def test_zero_rows_infinities_and_nan(N):
    x = torch.randn(6, N, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(N, dtype=torch.bfloat16, device="cuda")
    clean, clean_s = vig_b200.add_rmsnorm_8bit(x, w)
    x[1] = 0
    x[3, 7], x[4, 9] = float("nan"), float("inf")
    for out in (torch.float8_e4m3fn, torch.int8):
        q, s = vig_b200.add_rmsnorm_8bit(x, w, dtype=out)
        assert (q[1].float() == 0).all() and s[1] == 0
        assert torch.isnan(s[3]) and torch.isnan(s[4])
        assert torch.isfinite(s[[0, 2, 5]]).all()
        if out == torch.float8_e4m3fn:
            assert torch.equal(q[[0, 2, 5]].view(torch.uint8), clean[[0, 2, 5]].view(torch.uint8)) and torch.equal(s[[0, 2, 5]], clean_s[[0, 2, 5]])
    # an infinite weight: its channel takes the scale
    w[5] = float("inf")
    q, s = vig_b200.add_rmsnorm_8bit(x[:1], w)
    assert torch.isinf(s).all()
    # values whose scale would have no reciprocal count as zeros
    q, s = vig_b200.add_rmsnorm_8bit(torch.full((1, N), 1e-38, device="cuda"), torch.full((N,), 1e-3, device="cuda"), eps=1.0)
    assert (q.float() == 0).all() and (s == 0).all()


def test_strided_rows_and_leading_dimensions():
    wide = torch.randn(3, 5, 500, dtype=torch.float16, device="cuda")
    w = torch.randn(192, dtype=torch.float16, device="cuda")
    for lo in (0, 8, 3):
        x, res = wide[..., lo:lo + 192], wide.flip(0)[..., 200 + lo:392 + lo]
        for t in (x, x.transpose(0, 1)):
            rs = res if t is x else res.transpose(0, 1)
            a = vig_b200.add_rmsnorm_8bit(t, w, rs, prenorm=True)
            b = vig_b200.add_rmsnorm_8bit(t.contiguous(), w, rs.contiguous(), prenorm=True)
            assert a[1].shape == (*t.shape[:-1], 1)
            assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a, b))
    one = vig_b200.add_rmsnorm_8bit(wide[0, 0, :192], w)
    assert one[0].shape == (192,) and one[1].shape == (1,)
    # a row that is expanded over the batch
    rows = vig_b200.add_rmsnorm_8bit(wide[:1, :1, :192].expand(4, 1, 192), w)
    assert all(torch.equal(rows[0][i].view(torch.uint8), rows[0][0].view(torch.uint8)) for i in range(4))


def check_train(M, N, dtype, residual, with_dr, w_dtype=None):
    x, w, res = make(M, N, dtype, seed=M + N, residual=residual, w_dtype=w_dtype)
    gen = torch.Generator().manual_seed(1)
    dy = torch.randn(M, N, generator=gen).to(dtype)
    dr = torch.randn(M, N, generator=gen).to(dtype) if with_dr else None
    leaf = [t.cuda().requires_grad_(True) for t in (x, w, res) if t is not None]
    y, r = vig_b200.add_rmsnorm_train(leaf[0], leaf[1], leaf[2] if residual else None, eps=EPS)
    outs, ds = ([y, r], [dy.cuda(), dr.cuda()]) if with_dr else ([y], [dy.cuda()])
    grads = torch.autograd.grad(outs, leaf, ds)
    rd, rstd, yd = formula(x, w, res)
    unit, tiny, rel = UNIT[dtype], TINY[dtype], rel_rstd(N) + 4 * U
    assert ((y.detach().double().cpu() - yd).abs() <= (unit * 1.01 + rel + U) * yd.abs() + tiny).all()
    assert ((r.detach().double().cpu() - rd).abs() <= (unit * 1.01 + U) * rd.abs() + tiny).all()
    # gradients are taken at the sum as it was rounded (by e of itself where there is a residual)
    e = unit if residual else 0.0
    t, xh = dy.double() * w.double(), rd * rstd
    mean_txh = (t * xh).mean(-1, keepdim=True)
    want = rstd * (t - xh * mean_txh)
    size = rstd * (t.abs() + xh.abs() * (t * xh).abs().mean(-1, keepdim=True))
    off = (3 * e + 4 * rel) * size
    if with_dr:
        if residual:
            want = want + dr.double()
        else:
            want, off = want + dr.double(), off + unit * (want.abs() + off)      # r is x: the framework adds two rounded gradients
    assert ((grads[0].double().cpu() - want).abs() <= off + unit * 1.01 * (want.abs() + off) + 2 * U * want.abs() + tiny).all()
    if residual:
        assert torch.equal(grads[0], grads[2])
    dw = (dy.double() * xh).sum(0)
    mag = (dy.double() * xh).abs().sum(0)
    wu = UNIT[w.dtype]
    assert grads[1].dtype == w.dtype
    assert ((grads[1].double().cpu() - dw).abs() <= (2 * e + rel + (M + 8) * U) * mag + 1.01 * wu * dw.abs() + TINY[w.dtype]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", WIDTHS)
def test_training(N, dtype):
    check_train(1, N, dtype, True, True)
    check_train(37, N, dtype, False, False)
    check_train(70, N, dtype, True, False, torch.float32)


@pytest.mark.parametrize("M,N,dtype", [(5000, 192, torch.bfloat16), (3001, 384, torch.float16), (2000, 768, torch.float32), (700, 2048, torch.bfloat16)])
def test_training_many_rows(M, N, dtype):
    check_train(M, N, dtype, True, True)
    check_train(M, N, dtype, False, True)


def test_backward_by_itself_and_strided_gradients():
    x, w, res = cuda(*make(40, 192, torch.bfloat16, 3, True))
    _, r = vig_b200.add_rmsnorm_train(x, w, res)
    dy = torch.randn(40, 400, dtype=torch.bfloat16, device="cuda")[:, 5:197]
    dr = torch.randn(192, 40, dtype=torch.bfloat16, device="cuda").t()
    a = vig_b200.add_rmsnorm_backward(dy, r, w, d_r=dr)
    b = vig_b200.add_rmsnorm_backward(dy.contiguous(), r, w, d_r=dr.contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    leaf = [t.clone().requires_grad_(True) for t in (x, w, res)]
    y, _ = vig_b200.add_rmsnorm_train(*leaf)
    y.sum().backward()                         # a gradient of stride 0
    ones = vig_b200.add_rmsnorm_backward(torch.ones_like(y), x, w, residual=res)         # the sum as the forward had it, in fp32
    assert torch.equal(leaf[0].grad, ones[0]) and torch.equal(leaf[1].grad, ones[1])


def test_gradient_against_differences():
    x, w, res = (t.cuda().requires_grad_(True) for t in make(6, 50, torch.float32, 5, True))
    wy, wr = torch.randn(6, 50, device="cuda").double(), torch.randn(6, 50, device="cuda").double()

    def value(*ins):
        y, r = vig_b200.add_rmsnorm_train(*ins)
        return (y.double() * wy).sum() + (r.double() * wr).sum()

    grads = torch.autograd.grad(value(x, w, res), (x, w, res))
    eps = 2.0 ** -6
    for i, grad in enumerate(grads):
        ins = [t.detach() for t in (x, w, res)]
        v = torch.randn_like(ins[i])
        ends = []
        for sign in (1, -1):
            moved = list(ins)
            moved[i] = ins[i] + sign * eps * v
            ends.append(float(value(*moved)))
        # rounding of the values over the step: U / eps of their sum; the norm's third derivative by eps^2
        size = float((grad.double() * v).abs().sum()) + float(wy.abs().sum())
        assert abs((ends[0] - ends[1]) / (2 * eps) - float((grad.double() * v).sum())) <= (4 * U / eps + 4 * eps ** 2) * size


def test_same_bits_twice():
    x, w, res = cuda(*make(3000, 192, torch.bfloat16, 8, True))
    dy = torch.randn_like(x)
    _, r = vig_b200.add_rmsnorm_train(x, w, res)
    a, b = (vig_b200.add_rmsnorm_backward(dy, r, w) for _ in range(2))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_no_rows_and_refusals():
    x, w = torch.zeros(0, 64, device="cuda", requires_grad=True), torch.ones(64, device="cuda", requires_grad=True)
    q, s = vig_b200.add_rmsnorm_8bit(x, w)
    assert q.shape == (0, 64) and s.shape == (0, 1)
    y, _ = vig_b200.add_rmsnorm_train(x, w)
    y.sum().backward()
    assert x.grad.shape == (0, 64) and (w.grad == 0).all()
    x = torch.zeros(2, 64, device="cuda")
    w = w.detach()
    for bad in (lambda: vig_b200.add_rmsnorm_8bit(x, w[:32]), lambda: vig_b200.add_rmsnorm_8bit(x, w, x[:1]), lambda: vig_b200.add_rmsnorm_8bit(x, w, group=48),
                lambda: vig_b200.add_rmsnorm_8bit(x[:, :40], w[:40], group=32), lambda: vig_b200.add_rmsnorm_8bit(x, w, eps=-1.0),
                lambda: vig_b200.add_rmsnorm_train(x, w[None]), lambda: vig_b200.add_rmsnorm_8bit(x[:, :0], w[:0]), lambda: vig_b200.add_rmsnorm_backward(x[:1], x, w)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: vig_b200.add_rmsnorm_8bit(x, w.half()), lambda: vig_b200.add_rmsnorm_8bit(x, w, x.half()), lambda: vig_b200.add_rmsnorm_8bit(x, w, dtype=torch.float16),
                lambda: vig_b200.add_rmsnorm_train(x.double(), w.double()), lambda: vig_b200.add_rmsnorm_train(x, None)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: vig_b200.add_rmsnorm_8bit(x.cpu(), w), lambda: vig_b200.add_rmsnorm_train(x, w.cpu())):
        with pytest.raises(RuntimeError):
            bad()
    from vig_b200 import _lib
    L_ = _lib.lib()
    call = lambda rows=1, N=64, group=0, dtype=0, wd=0, out=0: L_.vig_add_rmsnorm_8bit_fwd(None, 64, None, 0, None, wd, None, None, None, rows, N, group, 1e-6, out, dtype, None)  # noqa: E731
    assert call() == -1 and call(dtype=5) == -3 and call(wd=1) == -3 and call(rows=-1) == -2 and call(N=0) == -2 and call(rows=0) == 0
    assert call(rows=0, group=48) == -2 and call(rows=0, out=2) == -6


@pytest.mark.parametrize("out", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("N", [192, 193, 20000])
def test_small_scales(N, out):
    """Rows whose scale is hardly above the smallest normal number, though the norm lifts them by a thousand."""
    top = 448 if out == torch.float8_e4m3fn else 127
    x = torch.full((1, N), 2.0 ** -30)
    x[0, ::2] = 0
    w = torch.full((N,), 2.0 ** -126 * top * 2.0 ** 21)       # y up to 1.5 times the smallest normal scale's range
    q, s = vig_b200.add_rmsnorm_8bit(x.cuda(), w.cuda(), eps=1e-6, dtype=out)
    assert 1.17549435e-38 <= float(s) < 2.4e-38
    assert (q[0, ::2].float() == 0).all() and (q[0, 1::2].float() == top).all()


def test_gradient_of_small_rows_without_eps():
    """eps = 0 and rows of 1e-15: rstd is 1e15 and its cube out of range, the gradient is not."""
    x, w, _ = make(3, 64, torch.float32, 4, False)
    x, dy = x * 1e-15, torch.randn(3, 64, generator=torch.Generator().manual_seed(6))
    dx, dw = vig_b200.add_rmsnorm_backward(dy.cuda(), x.cuda(), w.cuda(), eps=0.0)
    r = x.double()
    rstd = r.square().mean(-1, keepdim=True).rsqrt()
    t, xh = dy.double() * w.double(), r * rstd
    m = (t * xh).mean(-1, keepdim=True)
    rel = rel_rstd(64) + 4 * U
    assert ((dx.cpu().double() - rstd * (t - xh * m)).abs() <= 4 * rel * rstd * (t.abs() + xh.abs() * (t * xh).abs().mean(-1, keepdim=True))).all()
    assert ((dw.cpu().double() - (dy.double() * xh).sum(0)).abs() <= (rel + 16 * U) * (dy.double() * xh).abs().sum(0)).all()


def test_offsets_beyond_32_bits():
    """More than 2^31 values: the last rows as a call on them alone gives them, bit for bit (a row's arithmetic does not depend on its place)."""
    M, N = 2_900_000, 768
    gen = torch.Generator(device="cuda").manual_seed(8)
    x, res = (torch.empty(M, N, dtype=torch.bfloat16, device="cuda").normal_(generator=gen) for _ in range(2))
    w = torch.ones(N, dtype=torch.bfloat16, device="cuda")
    got, ref = vig_b200.add_rmsnorm_8bit(x, w, res, prenorm=True), vig_b200.add_rmsnorm_8bit(x[-40:], w, res[-40:], prenorm=True)
    assert all(torch.equal(a[-40:].view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, ref))
    dx, _ = vig_b200.add_rmsnorm_backward(x, got[2], w)
    assert torch.equal(dx[-40:], vig_b200.add_rmsnorm_backward(x[-40:], got[2][-40:], w)[0])
