"""The longest sums of the product of 8-bit integers: codes may be -128, so 131071 products of two are what a signed sum of 32 bits holds, and 131072 are refused."""
import pytest
import torch

import vig_b200
from vig_b200 import _lib

MOST = 131071


def test_entries():
    L_ = _lib.lib()
    mul = lambda K: L_.vig_linear_int8_fwd(None, K, None, None, K, None, None, None, 8, 1, 8, K, 0, None, None)  # noqa: E731
    assert mul(MOST) == -1 and mul(MOST + 1) == -2                             # NULL; too long
    assert L_.vig_int8_rows_lay_out(None, MOST, None, 1, MOST, None) == -1 and L_.vig_int8_rows_lay_out(None, MOST + 1, None, 1, MOST + 1, None) == -2
    # laid out, a row is no longer than the longest either
    first = lambda K: L_.vig_linear_int8_laid_out_first(257, K, 256, K, 4096, 256, K)  # noqa: E731
    assert first(131055) == 1 and first(131056) == 1 and first(131057) == 0 and first(MOST) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("K", [131055, 131056, 131057, MOST])
@pytest.mark.parametrize("M", [1, 9, 70])
def test_all_at_the_lowest_code(M, K):
    """2^14 K and -127 * 2^7 K, exactly: their 31 bits are one rounding to fp32."""
    q, w = torch.full((M, K), -128, dtype=torch.int8, device="cuda"), torch.full((20, K), -128, dtype=torch.int8, device="cuda")
    w[1::2] = 127
    y = vig_b200.linear_int8(q, torch.ones(M, 1, device="cuda"), w, torch.ones(20, device="cuda"), dtype=torch.float32)
    assert (y[:, ::2] == torch.tensor(2.0 ** 14 * K).float().item()).all() and (y[:, 1::2] == torch.tensor(-127.0 * 128 * K, dtype=torch.float64).float().item()).all()


@pytest.mark.gpu
def test_longer_rows_are_refused():
    q = torch.zeros(2, MOST + 1, dtype=torch.int8, device="cuda")
    with pytest.raises(ValueError, match="131071"):
        vig_b200.linear_int8(q, torch.ones(2, 1, device="cuda"), q, torch.ones(2, device="cuda"))
