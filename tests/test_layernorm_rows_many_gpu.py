"""The trainable layer norm over more rows than its threads: each takes several, with the next under way, and keeps its shares of the weight's and the bias's gradients from row to
row.  Reference and bounds as in test_layernorm_rows_gpu.py, evaluated on the GPU."""
import pytest
import torch

import vig_b200
from test_layernorm_rows_gpu import EPS, U, UNIT, reference

pytestmark = pytest.mark.gpu

# rows of 4, 16, 128 and 256 threads, whole vectors and not, and past what a block's threads hold: more of each than there are threads for at once
CASES = [(160001, 7, torch.bfloat16), (200704, 96, torch.bfloat16), (100003, 36, torch.float32), (40001, 333, torch.float16), (6001, 768, torch.float32), (5003, 2049, torch.float16),
         (3001, 4096, torch.float32), (3001, 8192, torch.bfloat16), (2501, 16392, torch.bfloat16), (2501, 9001, torch.float32)]


@pytest.mark.parametrize("M,N,dtype", CASES)
def test_many_rows(M, N, dtype):
    k = CASES.index((M, N, dtype))
    gen = torch.Generator(device="cuda").manual_seed(k)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    param = torch.float32 if k % 3 == 1 else dtype
    t = dict(x=(rand(M, N) + 0.5).to(dtype), weight=(1 + 0.2 * rand(N)).to(param), bias=rand(N).to(param), residual=(2 * rand(M, N)).to(dtype))
    d_y, d_r = rand(M, N).to(dtype), rand(M, N).to(dtype)
    leaf = {n: v.requires_grad_(True) for n, v in t.items()}
    y, r = vig_b200.add_layernorm_train(**leaf, eps=EPS)
    outs = [y, r, *torch.autograd.grad([y, r], list(leaf.values()), [d_y, d_r])]
    assert torch.equal(outs[2], outs[5])
    zeros = lambda v: torch.zeros(N, device="cuda", dtype=torch.float64)  # noqa: E731
    dw, e_w, db, e_b = (zeros(None) for _ in range(4))
    with torch.no_grad():
        # a few thousand rows of the reference at a time; their shares of the sums over all rows are added
        step = max(1, 2 ** 23 // N)
        for i in range(0, M, step):
            rows = slice(i, i + step)
            part = {n: v.detach() if n in ("weight", "bias") else v.detach()[rows] for n, v in t.items()}
            want = reference(part, d_y[rows], d_r[rows])
            for got, (ref, bound), what in zip((y[rows], r[rows], outs[2][rows]), want, ("y", "r", "dx")):
                most = bound + UNIT[dtype] * (ref.abs() + bound) + 2.0 ** -24
                off = (got.double() - ref).abs()
                assert (off <= most).all(), f"{what} from row {i}: worst {float((off / most).max()):.2f} of the bound"
            dw, e_w, db, e_b = dw + want[3][0], e_w + want[3][1], db + want[4][0], e_b + want[4][1]
            g = d_y[rows].double()
            xh = (want[0][0] - t["bias"].detach().double()) / t["weight"].detach().double()
            # the sums over all M rows round M times where those of a part rounded as often as it has rows
            e_w, e_b = e_w + (M - g.shape[0]) * U * (g * xh).abs().sum(0), e_b + (M - g.shape[0]) * U * g.abs().sum(0)
    for got, ref, bound, what in ((outs[3], dw, e_w, "dw"), (outs[4], db, e_b, "db")):
        most = bound + UNIT[param] * (ref.abs() + bound) + 2.0 ** -24
        off = (got.double() - ref).abs()
        assert torch.isfinite(got).all() and (off <= most).all(), f"{what}: worst {float((off / most).max()):.2f} of the bound"
        # that bound grows with M; errors of single rows, independent ones, with its root: no share may be missing or taken twice
        assert float((got.double() - ref).norm() / ref.norm()) < UNIT[param] + 64 * U * M ** 0.5
