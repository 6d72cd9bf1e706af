"""Products of 8-bit integers: sums are exact, so what is left is scaling.  With u = 2^-24: the integer's rounding to fp32, the product of the scales, their product with it and
the sum with the bias: 4 u of the sum of magnitudes, and the rounding to the output's type."""
import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
UNIT = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(M, N, K, dtype, seed, bias=True, full=False):
    gen = torch.Generator().manual_seed(seed)
    codes = lambda r: torch.full((r, K), -128, dtype=torch.int8) if full else torch.randint(-128, 128, (r, K), generator=gen, dtype=torch.int8)  # noqa: E731
    return codes(M), torch.rand(M, 1, generator=gen) * 1e-2, codes(N), torch.rand(N, generator=gen) * 1e-2, torch.randn(N, generator=gen).to(dtype) if bias else None


def check(got, q, s, w, ws, b, dtype):
    # (products of two bytes, up to 2^17 of them: below 2^53)
    value = (q.double() @ w.double().t()) * s.double() * ws.double()
    ref = value + (b.double() if b is not None else 0)
    bound = 4 * U * (value.abs() + (b.double().abs() if b is not None else 0))
    off = (got.double().cpu() - ref).abs()
    most = bound + UNIT[dtype] * (ref.abs() + bound) + 2.0 ** -24
    assert got.dtype == dtype and got.shape == ref.shape
    assert (off <= most).all(), f"worst {float((off / most).max()):.2f} of the bound"


SHAPES = [(1, 1, 1), (1, 16, 16), (3, 17, 15), (8, 192, 64), (8, 2304, 768), (9, 100, 80), (17, 33, 48), (33, 70, 272), (64, 192, 2064), (65, 64, 64), (100, 300, 33), (257, 257, 128), (300, 193, 144),
          (511, 40, 784), (1000, 576, 192), (130, 2304, 768), (70, 8, 16), (128, 1, 32)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(M, N, K, dtype):
    q, s, w, ws, b = make(M, N, K, dtype, seed=M + N + K, bias=(M + N) % 2 == 0)
    got = vig_b200.linear_int8(q.cuda(), s.cuda(), w.cuda(), ws.cuda(), None if b is None else b.cuda(), dtype=dtype)
    check(got, q, s, w, ws, b, dtype)


def test_rows_off_16_bytes():
    """Large products of rows that begin anywhere are taken over copies of them: odd K, and even ones behind an odd offset; K next to the largest is taken as it lies."""
    for M, N, K, first in ((5000, 300, 333, 0), (700, 96, 768, 3), (40, 2304, 767, 1), (300, 64, 131071, 0)):
        q, s, w, ws, b = make(M, N, K, torch.bfloat16, seed=K)
        wide = torch.zeros(M, K + first, dtype=torch.int8, device="cuda")
        wide[:, first:] = q.cuda()
        got = vig_b200.linear_int8(wide[:, first:], s.cuda(), w.cuda(), ws.cuda(), b.cuda())
        check(got, q, s, w, ws, b, torch.bfloat16)


def test_many_tiles():
    """More tiles than CTA pairs, W's columns stationary and streamed."""
    for M, N, K in ((20000, 768, 768), (40000, 300, 256), (3000, 2304, 2048)):
        q, s, w, ws, b = make(M, N, K, torch.bfloat16, seed=K)
        got = vig_b200.linear_int8(q.cuda(), s.cuda(), w.cuda(), ws.cuda(), b.cuda())
        rows = torch.randint(0, M, (300,), generator=torch.Generator().manual_seed(0))
        check(got[rows.cuda()], q[rows], s[rows], w, ws, b, torch.bfloat16)
        assert torch.isfinite(got).all()


def test_largest_sums():
    """All codes -128: 2^14 K, the largest a sum of 32 bits has to hold."""
    for M in (1, 70):
        q, s, w, ws, b = make(M, 20, 131056, torch.float32, seed=1, full=True)
        check(vig_b200.linear_int8(q.cuda(), s.cuda(), w.cuda(), ws.cuda(), b.cuda(), dtype=torch.float32), q, s, w, ws, b, torch.float32)


def test_views_and_shapes():
    """Rows of wider matrices on 16 bytes and off them, and leading dimensions; every form of the kernel gives the same bits."""
    for M in (12, 150):
        q, s, w, ws, b = (t.cuda() for t in make(M, 48, 80, torch.bfloat16, seed=5))
        plain = vig_b200.linear_int8(q, s, w, ws, b)
        for first in (0, 16, 3):
            wide_q, wide_w = torch.zeros(M, 128, dtype=torch.int8, device="cuda"), torch.zeros(48, 112, dtype=torch.int8, device="cuda")
            wide_q[:, first:first + 80], wide_w[:, first:first + 80] = q, w
            assert torch.equal(vig_b200.linear_int8(wide_q[:, first:first + 80], s, wide_w[:, first:first + 80], ws, b), plain)
        y = vig_b200.linear_int8(q.view(M // 6, 2, 3, 80), s.view(M // 6, 2, 3), w, ws[:, None], b)
        assert y.shape == (M // 6, 2, 3, 48) and torch.equal(y.view(M, 48), plain)


def test_behind_a_quantizing_norm():
    """What add_rmsnorm_8bit leaves goes straight in: the product is the one of the rows it stands for."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    for M in (5, 200):
        x, g = torch.randn(M, 192, generator=gen, device="cuda").bfloat16(), torch.ones(192, device="cuda").bfloat16()
        q, s = vig_b200.add_rmsnorm_8bit(x, g, dtype=torch.int8)
        w = torch.randint(-127, 128, (576, 192), generator=gen, device="cuda", dtype=torch.int8)
        ws = torch.rand(576, generator=gen, device="cuda") * 1e-2
        check(vig_b200.linear_int8(q, s, w, ws), q.cpu(), s.cpu(), w.cpu(), ws.cpu(), None, torch.bfloat16)


def test_far_rows():
    q, s, w, ws, b = (t.cuda() for t in make(70, 32, 64, torch.bfloat16, seed=2))
    far = torch.empty(70 * 2 ** 25 + 64, dtype=torch.int8, device="cuda").as_strided((70, 64), (2 ** 25, 1))
    far.copy_(q)
    assert torch.equal(vig_b200.linear_int8(far, s, w, ws, b), vig_b200.linear_int8(q, s, w, ws, b))
    assert torch.equal(vig_b200.linear_int8(far[:9], s[:9], w, ws, b), vig_b200.linear_int8(q[:9], s[:9], w, ws, b))


def test_graph_and_stream():
    for M in (8, 300):
        q, s, w, ws, b = (t.cuda() for t in make(M, 96, 192, torch.bfloat16, seed=3))
        plain = vig_b200.linear_int8(q, s, w, ws, b)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        other = torch.zeros_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = vig_b200.linear_int8(other, s, w, ws, b)
        other.copy_(q)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, plain)
    vig_b200.check_status()


def test_empty_and_refusals():
    q, s, w, ws, b = (t.cuda() for t in make(4, 8, 16, torch.bfloat16, seed=0))
    assert vig_b200.linear_int8(q[:0], s[:0], w, ws).shape == (0, 8) and vig_b200.linear_int8(q, s, w[:0], ws[:0]).shape == (4, 0)
    assert torch.equal(vig_b200.linear_int8(q[:, :0], s, w[:, :0], ws, b), b.expand(4, 8))
    call = lambda **kw: vig_b200.linear_int8(**{**dict(q=q, scales=s, weight=w, weight_scales=ws, bias=b), **kw})  # noqa: E731
    for bad in (dict(q=q[:, :15]), dict(scales=s[:3]), dict(weight_scales=ws[:7]), dict(bias=b[:7]), dict(weight=w.t()), dict(scales=s.t())):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(q=q.to(torch.uint8)), dict(weight=w.float()), dict(scales=s.half()), dict(bias=b.float()), dict(dtype=torch.float64)):
        with pytest.raises(TypeError):
            call(**bad)
    with pytest.raises(NotImplementedError):
        call(scales=s.clone().requires_grad_(True))
