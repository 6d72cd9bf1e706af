"""What the operators of a block with a selective state space refuse without a GPU: tensors of the CPU, and at the C entry points every argument that is looked at before
anything is launched."""
import ctypes

import pytest
import torch

import vig_b200
from vig_b200 import _lib

X, W, V = torch.zeros(2, 4, 8), torch.zeros(8, 4), torch.ones(8)


@pytest.mark.parametrize("call", [
    lambda: vig_b200.selective_scan(X, X, W, X, X),
    lambda: vig_b200.selective_scan_step(X[:, 0], X[:, 0], W, X[:, 0], X[:, 0], torch.zeros(2, 8, 4)),
    lambda: vig_b200.causal_conv(X, W),
    lambda: vig_b200.causal_conv_step(X[:, 0], torch.zeros(2, 3, 8), W),
    lambda: vig_b200.add_layernorm_train(X, V),
    lambda: vig_b200.add_layernorm_backward(X, X, V),
    lambda: vig_b200.linear_int8(X.to(torch.int8), X[..., :1], W.t().to(torch.int8), V[:4]),
], ids=["scan", "scan_step", "conv", "conv_step", "norm", "norm_backward", "int8"])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="CUDA"):
        call()


def test_arguments_that_python_looks_at():
    with pytest.raises(ValueError, match="activation"):
        vig_b200.causal_conv(X, W, activation="gelu")
    with pytest.raises(TypeError):
        vig_b200.linear_int8(X, X, W, V, dtype=torch.int32)


class Args(ctypes.Structure):
    """vig_selective_scan_args"""
    _fields_ = ([(n, ctypes.c_int32) for n in ("B", "L", "D", "N", "G", "dtype", "skip_dtype", "bias_dtype", "softplus", "reserved")] +
                [(n, ctypes.c_void_p) for n in ("u", "dt", "z", "b", "c", "A", "skip", "dt_bias", "lengths", "h0")] + [("ld_h0", ctypes.c_int64)] +
                [(n, ctypes.c_void_p) for n in ("y", "h_final")] + [("ld_final", ctypes.c_int64), ("states", ctypes.c_void_p)] +
                [("strides", ctypes.c_int64 * 14)] + [("d_y", ctypes.c_void_p), ("s_dy", ctypes.c_int64 * 2)] +
                [(n, ctypes.c_void_p) for n in ("d_final", "d_u", "d_dt", "d_z", "d_b", "d_c", "d_A", "d_skip", "d_bias", "d_h0", "workspace")] +
                [("workspace_bytes", ctypes.c_size_t), ("status", ctypes.c_void_p)])


def test_scan_entries():
    L_ = _lib.lib()
    base = dict(B=1, L=4, D=8, N=16, G=1)
    fwd = lambda **kw: L_.vig_selective_scan_fwd(ctypes.byref(Args(**{**base, **kw})), None)  # noqa: E731
    assert L_.vig_selective_scan_fwd(None, None) == -1 and fwd() == -1
    assert fwd(dtype=3) == -3 and fwd(dtype=-1) == -3 and fwd(dtype=1, skip=16, skip_dtype=2) == -3 and fwd(dt_bias=16, bias_dtype=7) == -3
    for bad in (dict(B=-1), dict(L=-1), dict(D=-1), dict(N=0), dict(N=65), dict(G=0), dict(G=3), dict(L=1 << 30), dict(B=1 << 16, D=1 << 15)):
        assert fwd(**bad) == -2, bad
    assert fwd(B=0) == 0 and fwd(D=0) == 0
    bwd = lambda **kw: L_.vig_selective_scan_bwd(ctypes.byref(Args(**{**base, **kw})), None)  # noqa: E731
    assert bwd() == -1 and bwd(N=65) == -2 and bwd(B=0) == 0
    step = lambda **kw: L_.vig_selective_scan_step(ctypes.byref(Args(**{**base, "L": 1, **kw})), None)  # noqa: E731
    assert step() == -1 and step(L=2) == -2 and step(N=0) == -2 and step(B=0) == 0
    everything = {n: 256 for n in ("u", "dt", "b", "c", "A", "states", "d_y", "d_u", "d_dt", "d_b", "d_c", "d_A")}
    assert bwd(**everything) == -5                                            # no workspace
    assert L_.vig_selective_scan_states_bytes(2, 65, 8, 16) == 2 * 2 * 8 * 16 * 4 and L_.vig_selective_scan_states_bytes(0, 65, 8, 16) == 0
    assert L_.vig_selective_scan_bwd_workspace_bytes(1, 4, 8, 16, 1) >= 4 * (2 * 4 * 16 + 8 * 18) and L_.vig_selective_scan_bwd_workspace_bytes(1, 4, 8, 16, 0) == 0


def test_conv_entries():
    L_ = _lib.lib()
    fwd = lambda B=1, L=4, D=8, K=4, wd=0, dtype=0: L_.vig_causal_conv_fwd(None, None, wd, None, None, None, None, None, B, L, D, K, None, None, None, None, 0, dtype, None)  # noqa: E731
    assert fwd() == -1 and fwd(dtype=4) == -3 and fwd(wd=1) == -3 and fwd(K=0) == -2 and fwd(K=9) == -2 and fwd(B=-1) == -2 and fwd(L=1 << 30) == -2
    assert fwd(B=0) == 0 and fwd(D=0) == 0 and fwd(L=0) == 0
    bwd = lambda **kw: L_.vig_causal_conv_bwd(None, 256, 0, None, None, None, None, None, None, 256, None, None, kw.get("B", 1), kw.get("L", 0), 8, kw.get("K", 4), None, None, None, 0, 0, None, 0, None)  # noqa: E731
    assert bwd() == -5 and bwd(L=4) == -1 and bwd(K=9) == -2 and bwd(B=0) == 0
    assert L_.vig_causal_conv_step(None, 8, None, None, None, 0, None, None, 8, 1, 8, 4, 0, 0, None) == -1
    assert L_.vig_causal_conv_step(None, 8, None, None, None, 0, None, None, 8, 0, 8, 4, 0, 0, None) == 0
    assert L_.vig_causal_conv_bwd_workspace_bytes(0, 4, 8, 4) == 0


def test_norm_and_product_entries():
    L_ = _lib.lib()
    fwd = lambda rows=1, N=64, wd=0, dtype=0: L_.vig_add_layernorm_train_fwd(None, N, None, 0, None, None, wd, None, None, rows, N, 1e-5, dtype, None)  # noqa: E731
    assert fwd() == -1 and fwd(dtype=5) == -3 and fwd(wd=1) == -3 and fwd(rows=-1) == -2 and fwd(N=0) == -2 and fwd(rows=0) == 0
    bwd = lambda **kw: L_.vig_add_layernorm_bwd(256, 8, 256, 8, None, 0, 256, 0, None, 0, 256, kw.get("dw", 256), None, 1, 8, 1e-5, 0, None, 0, None)  # noqa: E731
    assert bwd() == -5 and bwd(dw=None) == -1
    assert L_.vig_add_layernorm_bwd_workspace_bytes(0, 64) == 0 and L_.vig_add_layernorm_bwd_workspace_bytes(10, 64) >= 2 * 64 * 4
    mul = lambda M=1, N=8, K=16, dtype=0: L_.vig_linear_int8_fwd(None, K, None, None, K, None, None, None, N, M, N, K, dtype, None, None)  # noqa: E731
    assert mul() == -1 and mul(dtype=3) == -3 and mul(M=-1) == -2 and mul(K=131073) == -2 and mul(N=-1) == -2 and mul(M=0) == 0 and mul(N=0) == 0


def test_laying_out():
    L_ = _lib.lib()
    first = lambda x=256, ldx=64, M=4096, N=256, K=64: L_.vig_linear_int8_laid_out_first(x, ldx, 256, 64, M, N, K)  # noqa: E731
    assert first() == 0 and first(x=257) == 1 and first(ldx=65) == 1 and first(K=63) == 1 and first(K=63, M=4) == 0 and first(M=0) == 0 and first(K=131071) == 0
    lay = lambda src=None, dst=None, rows=1, K=5: L_.vig_int8_rows_lay_out(src, 5, dst, rows, K, None)  # noqa: E731
    assert lay() == -1 and lay(rows=-1) == -2 and lay(K=131073) == -2 and lay(rows=0) == 0 and lay(K=0) == 0 and lay(src=256, dst=264) == -4


def test_block_refuses_what_it_cannot_do():
    block = vig_b200.SelectiveStateSpace(16)
    with pytest.raises(RuntimeError, match="CUDA"):
        block(torch.zeros(1, 3, 16))
    with pytest.raises(TypeError):
        vig_b200.GatedRecurrence(16).quantize(torch.int16)
