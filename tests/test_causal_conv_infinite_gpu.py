"""The causal convolution's weight gradient beside the end of a sequence: tokens behind it have no share, not even nothing times what stands in their windows."""
import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [12, 5])
@pytest.mark.parametrize("K", [2, 4, 8])
@pytest.mark.parametrize("end", [1, 7, 8, 19, 40])
def test_infinite_last_token(end, K, D, dtype):
    """An infinite last token meets the last tap alone: dw_k = sum over t < end of dy_t x_{t-K+1+k}, whole numbers and their sums exact."""
    gen = torch.Generator().manual_seed(end + K)
    whole = lambda *s: torch.randint(-2, 3, s, generator=gen).to(dtype).cuda()  # noqa: E731
    x, w, d = whole(2, 40, D), whole(D, K).requires_grad_(True), whole(2, 40, D)
    d[:, end - 1] = 1
    x[0, end - 1] = float("inf")
    lengths = torch.tensor([end, 40], device="cuda")
    y, _ = vig_b200.causal_conv(x, w, lengths=lengths)
    dw, = torch.autograd.grad(y, w, d)
    want = torch.zeros(D, K, dtype=torch.float64, device="cuda")
    for b, n in enumerate((end, 40)):
        for k in range(K - 1):
            at = slice(max(0, K - 1 - k), n)
            want[:, k] += (d[b, at].double() * x[b, max(0, K - 1 - k) - (K - 1 - k):n - (K - 1 - k)].double()).sum(0) if n > K - 1 - k else 0
    assert torch.equal(dw[:, :K - 1].double(), want[:, :K - 1].to(dtype).double()) and (dw[:, K - 1] == float("inf")).all()
