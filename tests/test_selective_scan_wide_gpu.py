"""The selective scan's training call in the forms that many channels take (8 or 16 channels a block of threads, 1, 2 or 4 warps), with all gradients, and its accuracy as a
norm.  Reference and bounds as in test_selective_scan_gpu.py."""
import pytest
import torch

from test_selective_scan_gpu import NAMES, U, compare, make, reference, run

pytestmark = pytest.mark.gpu

# on 148 SMs: 16 channels by 2, 2, 1, 4 and 4 warps; 8 channels by 4
WIDE = [(90, 100, 256, 5, torch.bfloat16), (40, 128, 256, 16, torch.float32), (80, 60, 256, 16, torch.float16), (20, 200, 256, 16, torch.bfloat16), (12, 130, 512, 8, torch.float32),
        (10, 130, 256, 16, torch.bfloat16)]


@pytest.mark.parametrize("B,L,D,N,dtype", WIDE)
def test_gradients_of_many_channels(B, L, D, N, dtype):
    k = WIDE.index((B, L, D, N, dtype))
    t = make(B, L, D, N, 2 if k == 4 else 0, dtype, seed=k, state=k % 2 == 0)
    lengths = torch.randint(0, L + 1, (B,), generator=torch.Generator().manual_seed(k), dtype=torch.int32) if k in (1, 3) else None
    outs = compare(t, lengths)
    with torch.no_grad():
        y, final = run(t, None if lengths is None else lengths.cuda())
    assert torch.equal(y, outs[0]) and torch.equal(final, outs[1])


@pytest.mark.parametrize("B,L,D,N", [(2, 63, 24, 16), (2, 130, 20, 8), (2, 200, 12, 20), (1, 200, 40, 16)])
def test_accuracy_of_fp32(B, L, D, N):
    """Relative norms of the differences.  With u = 2^-24 and independent roundings: up to 200 decays in a product, each off by 4 u at most, 4 sqrt(200) u = 57 u, once in a state
    and once more in what goes back; their exponents, rounded three times, 3 u s |x| of a product e^(-s |x|), which is small where s |x| is above 3: 9 u, twice; sums of up
    to 400 terms sqrt(400) u and three of N and D terms beside them, 40 u.  Together 172 u; 256 u is 1.5e-5.  One operand in 16 bits would be 2^-9 / sqrt(3), 75 times that."""
    t = make(B, L, D, N, 0, torch.float32, seed=L + N)
    gen = torch.Generator().manual_seed(0)
    d_y, d_f = torch.randn(B, L, D, generator=gen), torch.randn(B, D, N, generator=gen)
    ref, _, _ = reference(t, d_y, d_f)
    for name, got, want in zip(("y", "final", *NAMES), run(t, None, d_y, d_f), ref):
        off = float((got.detach().double().cpu() - want).norm() / want.norm())
        assert off < 256 * U, f"{name}: {off / U:.0f} u"
