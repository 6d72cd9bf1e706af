"""RMS norm rows: codes of NaN alike in every form, the backward's forms over several rows of a CTA, and its sum in fp32.

Tolerances as in test_rmsnorm_rows_gpu.py, but gradients of add_rmsnorm_train are taken at the sum in fp32 in every type: nothing is allowed for a
rounding of it."""
import pytest
import torch

import vig_b200
from test_rmsnorm_rows_gpu import EPS, TINY, U, UNIT, formula, rel_rstd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [64, 192, 193, 5000, 9000, 20000])
@pytest.mark.parametrize("group", [None, 32])
@pytest.mark.parametrize("out", [torch.int8, torch.float8_e4m3fn])
def test_codes_of_nan(N, group, out):
    """A row, or a group, with a NaN has the scale NaN; its codes are 0 in int8, and NaN in e4m3, whichever form takes the row."""
    if group and N % group:
        N -= N % group
    x = torch.randn(3, N, device="cuda").bfloat16()
    x[1, N // 2] = float("nan")
    q, s = vig_b200.add_rmsnorm_8bit(x, torch.ones(N, dtype=torch.bfloat16, device="cuda"), dtype=out, group=group)
    assert torch.isnan(s[1]).all() and torch.isfinite(s[[0, 2]]).all()
    assert (q[1] == 0).all() if out == torch.int8 else torch.isnan(q[1].float()).all()


def check(M, N, dtype, residual, w_dtype=None):
    gen = torch.Generator(device="cuda").manual_seed(M + N)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x, res = rand(M, N).to(dtype), (2 * rand(M, N)).to(dtype) if residual else None
    w, dy, dr = (1 + 0.3 * rand(N)).to(w_dtype or dtype), rand(M, N).to(dtype), rand(M, N).to(dtype)
    leaf = [t.clone().requires_grad_(True) for t in (x, w, res) if t is not None]
    y, r = vig_b200.add_rmsnorm_train(leaf[0], leaf[1], leaf[2] if residual else None, eps=EPS)
    grads = torch.autograd.grad([y, r], leaf, [dy, dr]) if residual else torch.autograd.grad(y, leaf, dy)
    rd, rstd, _ = formula(x, w, res)
    rel, unit = rel_rstd(N) + 4 * U, UNIT[dtype]
    t, xh = dy.double() * w.double(), rd * rstd
    want = rstd * (t - xh * (t * xh).mean(-1, keepdim=True)) + (dr.double() if residual else 0)
    off = 4 * rel * rstd * (t.abs() + xh.abs() * (t * xh).abs().mean(-1, keepdim=True))
    assert ((grads[0].double() - want).abs() <= off + unit * 1.01 * (want.abs() + off) + 2 * U * want.abs() + TINY[dtype]).all()
    terms = dy.double() * xh
    dw, mag = terms.sum(0), terms.abs().sum(0)
    bound = (rel + (M + 8) * U) * mag
    assert ((grads[1].double() - dw).abs() <= bound + 1.01 * UNIT[w.dtype] * dw.abs() + TINY[w.dtype]).all()
    rounded = formula((x + res if residual else x), w, None)          # the formula at the sum as its type holds it
    return grads[1].double() - dw, dw, bound, (dy.double() * rounded[0] * rounded[1]).sum(0) - dw


@pytest.mark.parametrize("M,N,dtype", [(700, 9000, torch.bfloat16), (400, 16384, torch.float16), (500, 8192, torch.float32), (450, 4097, torch.float32), (1300, 5000, torch.bfloat16),
                                       (3000, 193, torch.bfloat16), (20000, 64, torch.float16), (9000, 768, torch.bfloat16), (1000, 20001, torch.bfloat16)])
def test_rows_of_a_cta(M, N, dtype):
    """More rows than find room at once: rows ahead in shared memory, one and two of them, and the form for rows wider than registers."""
    check(M, N, dtype, True)
    check(M, N, dtype, False)


@pytest.mark.parametrize("N", [192, 768, 1000, 20000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weight_gradient_at_the_unrounded_sum(N, dtype):
    """With weights in fp32 the gradient of 64 rows is right to fp32's sums; the formula at the sum of x and residual rounded to 16 bits is further off
    than that, where rows are not so wide that the bound of rstd's sum is as large."""
    off, _, bound, rounded = check(64, N, dtype, True, torch.float32)
    assert float(off.norm()) <= float(bound.norm())
    if N <= 1000:
        assert float(rounded.norm()) > 2 * float(bound.norm())
