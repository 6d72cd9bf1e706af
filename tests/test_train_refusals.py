"""What the operators of a trained and served recurrent block refuse without a GPU: tensors of the CPU, and at the C entry points every argument
that is looked at before anything is launched."""
import ctypes

import pytest
import torch

import vig_b200
from vig_b200 import _lib

X, W, S = torch.zeros(2, 4, 8), torch.ones(8), torch.zeros(2, 8)


@pytest.mark.parametrize("call", [
    lambda: vig_b200.gated_recurrence(X, X),
    lambda: vig_b200.gated_recurrence_step(S, S, S),
    lambda: vig_b200.add_rmsnorm_8bit(X, W),
    lambda: vig_b200.add_rmsnorm_train(X, W),
    lambda: vig_b200.add_rmsnorm_backward(X, X, W),
    lambda: vig_b200.adamw_step([S], [S], [S], [S], 1),
], ids=["recurrence", "step", "norm8", "norm", "norm_backward", "adamw"])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="CUDA"):
        call()


def test_optimizer_refuses_what_it_cannot_do():
    p = torch.zeros(3, requires_grad=True)
    for kw in (dict(state_bits=4), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            vig_b200.AdamW([p], **kw)
    with pytest.raises(TypeError):
        vig_b200.add_rmsnorm_8bit(X, W, dtype=torch.float16)


def test_recurrence_entry():
    L_ = _lib.lib()
    call = lambda B=1, L=4, D=8, norm=0.0, dtype=0: L_.vig_gated_recurrence_fwd(None, None, None, 0, None, None, 0, B, L, D, None, None, None, norm, 0, dtype, None, None)  # noqa: E731
    assert call() == -1                                                       # NULL
    assert call(dtype=3) == -3 and call(dtype=-1) == -3
    assert call(B=-1) == -2 and call(L=-1) == -2 and call(L=1 << 30) == -2 and call(B=1 << 16, D=1 << 15) == -2
    assert call(norm=-1.0) == -6 and call(norm=float("nan")) == -6 and call(norm=float("inf")) == -6
    assert call(B=0) == 0 and call(L=0) == 0 and call(D=0) == 0                # nothing to do
    bwd = lambda L=4, dtype=0: L_.vig_gated_recurrence_bwd(None, None, None, None, None, None, None, None, 1, L, 8, None, None, None, 0.0, 0, dtype, None, None)  # noqa: E731
    assert bwd() == -1 and bwd(dtype=9) == -3 and bwd(L=0) == 0


def test_norm_entries():
    L_ = _lib.lib()
    fwd = lambda rows=1, N=64, group=0, dtype=0, wd=0, out=0: L_.vig_add_rmsnorm_8bit_fwd(None, N, None, 0, None, wd, None, None, None, rows, N, group, 1e-6, out, dtype, None)  # noqa: E731
    assert fwd() == -1 and fwd(dtype=5) == -3 and fwd(wd=1) == -3 and fwd(rows=-1) == -2 and fwd(N=0) == -2
    assert fwd(rows=0) == 0 and fwd(rows=0, group=48) == -2 and fwd(rows=0, N=40, group=32) == -2 and fwd(rows=0, out=2) == -6
    assert L_.vig_add_rmsnorm_train_fwd(None, 8, None, 0, None, 0, None, None, 1, 8, 1e-6, 0, None) == -1
    assert L_.vig_add_rmsnorm_bwd(None, 8, None, 8, None, 0, None, 0, None, 0, None, None, 1, 8, 1e-6, 0, None, 0, None) == -1
    assert L_.vig_add_rmsnorm_bwd_workspace_bytes(0, 64) == 0 and L_.vig_add_rmsnorm_bwd_workspace_bytes(10, 64) >= 64 * 4


def test_adamw_entry():
    L_ = _lib.lib()
    one = (ctypes.c_void_p * 1)()
    n, code = (ctypes.c_int64 * 1)(4), (ctypes.c_int * 1)(0)

    def call(count=1, ptrs=one, numels=n, codes=code, step=1, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0):
        return L_.vig_adamw_step(count, ptrs, ptrs, ptrs, ptrs, None, None, None, numels, codes, codes, step, lr, b1, b2, eps, wd, None, None, None)

    assert call() == -1 and call(ptrs=None) == -1                              # a tensor of four values at NULL; no tables
    assert call(count=0) == 0 and call(numels=(ctypes.c_int64 * 1)(0)) == 0    # nothing to do
    assert call(numels=(ctypes.c_int64 * 1)(-1)) == -2 and call(numels=(ctypes.c_int64 * 1)(0), codes=(ctypes.c_int * 1)(7)) == -3
    for bad in (dict(step=0), dict(lr=-1.0), dict(lr=float("nan")), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(wd=-1.0), dict(count=-1)):
        assert call(**bad) == -6, bad
