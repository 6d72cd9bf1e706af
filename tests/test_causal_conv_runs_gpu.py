"""The short causal convolution over calls so large that a thread's run of tokens is many blocks long: blocks under way in a ring that is used again and again, long stretches
inside a sequence, and the borders of runs.  Reference and bounds as in test_causal_conv_gpu.py, for channels at both ends, which know nothing of the others."""
import pytest
import torch

import vig_b200
from test_causal_conv_gpu import check, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,L,D,K,state,ragged", [(64, 1021, 768, 4, True, False), (64, 1021, 765, 4, False, False), (64, 1021, 768, 4, True, True), (48, 1021, 765, 3, True, True),
                                                   (16, 2050, 768, 8, True, False), (3, 20011, 96, 5, True, True), (40, 2047, 512, 1, False, True)])
def test_long_runs(B, L, D, K, state, ragged, dtype):
    t = make(B, L, D, K, dtype, seed=L + D + K, state=state, param=torch.float32 if K == 8 else None)
    gen = torch.Generator().manual_seed(1)
    d_y, d_f = torch.randn(B, L, D, generator=gen).to(dtype), torch.randn(B, K - 1, D, generator=gen).to(dtype)
    n = None
    if ragged:
        n = torch.randint(0, L + 1, (B,), generator=gen, dtype=torch.int32)
        n[:3] = torch.tensor([L, 0, L - 1])
    leaf = {k: None if v is None else v.cuda().requires_grad_(True) for k, v in t.items()}
    names = [k for k, v in leaf.items() if v is not None]
    lengths = None if n is None else n.cuda()

    def call():
        y, final = vig_b200.causal_conv(**leaf, output_final_state=True, activation="silu", lengths=lengths)
        return [y, final, *torch.autograd.grad([y, final], [leaf[k] for k in names], [d_y.cuda(), d_f.cuda()])]

    outs = call()
    assert all(torch.equal(a, b) for a, b in zip(outs, call()))
    for at in (slice(0, 6), slice(D // 2 - 1, D // 2 + 5), slice(D - 6, D)):
        some = {k: None if v is None else v[at] if k in ("weight", "bias") else v[..., at] for k, v in t.items()}
        want = dict(zip(("y", "final", *t), reference(some, True, d_y[..., at], d_f[..., at], n)))
        for what, o in zip(("y", "final", *names), outs):
            check(o[at] if what in ("weight", "bias") else o[..., at], want[what], what)
