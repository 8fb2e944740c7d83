"""Refusals of the feed-forward block's operators that need no GPU: the Python wrappers'
messages and the C entry points' argument checks, which all return before any CUDA call."""

from __future__ import annotations

import ctypes

import pytest
import torch

import cuda_force_b200 as cf
from cuda_force_b200 import _abi

F = ctypes.c_void_p(0x1000)
BF16, F16, F32 = _abi.CF_DTYPE_BF16, _abi.CF_DTYPE_F16, _abi.CF_DTYPE_F32


def test_gated_residual_rmsnorm_refuses():
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    call = cf.gated_residual_rmsnorm
    with pytest.raises(ValueError, match="same shape"):
        call(x, torch.zeros(2, 3, 9), w)
    with pytest.raises(ValueError, match="share one dtype"):
        call(x, x.half(), w)
    with pytest.raises(ValueError, match="share one dtype"):
        call(x.double(), x.double(), w)
    with pytest.raises(ValueError, match="^weight must be 1-D of length 8"):
        call(x, x, torch.ones(9))
    with pytest.raises(ValueError, match="post_weight must be 1-D of length 8"):
        call(x, x, w, torch.ones(1, 8))
    with pytest.raises(ValueError, match="residual_scale must be a number"):
        call(x, x, w, residual_scale=torch.ones((), requires_grad=True))
    for bad in ((9,), (1, 3, 8), (3, 8), (2, 1, 1), (2, 2, 8)):
        with pytest.raises(ValueError, match="gate must be"):
            call(x, x, w, None, torch.ones(bad))
    for fine in ((8,), (1, 1, 8), (2, 1, 8), (2, 3, 8)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call(x, x, w, None, torch.ones(fine))


def test_gated_residual_rmsnorm_entry_points_refuse():
    lib = _abi.load()

    def fwd(rows=4, cols=64, groups=1, gate=F, x=F, dt=BF16, wdt=BF16):
        return lib.cf_gated_residual_rmsnorm(x, F, F, F, gate, groups, wdt, F, F, None, rows, cols,
                                             1.0, 1e-6, dt, None)

    assert fwd(rows=-1) == _abi.CF_ERR_INVALID_ARGUMENT
    assert fwd(cols=-1) == _abi.CF_ERR_INVALID_ARGUMENT
    assert fwd(groups=0) == _abi.CF_ERR_INVALID_ARGUMENT
    assert fwd(groups=3) == _abi.CF_ERR_INVALID_ARGUMENT
    assert fwd(x=None) == _abi.CF_ERR_INVALID_ARGUMENT
    assert fwd(dt=7) == _abi.CF_ERR_UNSUPPORTED
    assert fwd(wdt=F16) == _abi.CF_ERR_UNSUPPORTED
    assert fwd(rows=1 << 32) == _abi.CF_ERR_INVALID_ARGUMENT
    assert fwd(rows=0) == _abi.CF_OK
    assert fwd(cols=0) == _abi.CF_OK

    size = lib.cf_gated_residual_rmsnorm_backward_workspace_bytes
    assert size(0, 64, 1, 0, BF16) == 0 and size(4, 64, 1, 3, BF16) == 0
    assert size(1 << 20, 4096, 1, 1, BF16) < 1 << 28

    def bwd(rows=4, post=F, dpost=F, gate=F, dgate=F, stats=F, ws=F, ws_bytes=1 << 30):
        return lib.cf_gated_residual_rmsnorm_backward(
            F, F, F, F, F, post, gate, 1, BF16, stats, F, F, F, dpost, dgate, rows, 64, 1.0, BF16,
            ws, ws_bytes, None)

    assert bwd(dpost=None) == _abi.CF_ERR_INVALID_ARGUMENT
    assert bwd(gate=None) == _abi.CF_ERR_INVALID_ARGUMENT
    assert bwd(stats=None) == _abi.CF_ERR_INVALID_ARGUMENT
    assert bwd(ws=None) == _abi.CF_ERR_WORKSPACE
    assert bwd(ws_bytes=16) == _abi.CF_ERR_WORKSPACE
    assert bwd(ws=ctypes.c_void_p(0x1008)) == _abi.CF_ERR_MISALIGNED
    assert bwd(rows=0) == _abi.CF_OK


def test_fp8_wrappers_refuse():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    codes = torch.zeros(300, 256, dtype=torch.float8_e4m3fn)
    scales = torch.ones(3, 2)
    with pytest.raises(ValueError, match="block_rows must be 1 or 128"):
        cf.quantize_fp8(x, 64)
    with pytest.raises(ValueError, match="2-D for square blocks"):
        cf.quantize_fp8(x.view(2, 2, 256), 128)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        cf.quantize_fp8(x.double())
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        cf.linear_fp8(x, torch.zeros(300, 256, dtype=torch.int8), scales)
    with pytest.raises(ValueError, match="block scales"):
        cf.linear_fp8(x, codes, torch.ones(300, 2))
    with pytest.raises(ValueError, match="block scales"):
        cf.linear_fp8(x, codes, scales.double())
    with pytest.raises(ValueError, match="input features"):
        cf.linear_fp8(x[:, :128], codes, scales)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        cf.linear_fp8(x.float(), codes, scales)
    a = codes[:4]
    with pytest.raises(ValueError, match="block scales"):
        cf.matmul_fp8(a, torch.ones(1, 2), codes, scales)
    with pytest.raises(ValueError, match="input features"):
        cf.matmul_fp8(a[:, :128], torch.ones(4, 1), codes, scales)
    with pytest.raises(ValueError, match="returns float16 or bfloat16"):
        cf.matmul_fp8(a, torch.ones(4, 2), codes, scales, torch.float32)
    with pytest.raises(RuntimeError, match="CUDA"):
        cf.linear_fp8(x, codes, scales)
    with pytest.raises(RuntimeError, match="CUDA"):
        cf.quantize_fp8(x)


def test_fp8_entry_points_refuse():
    lib = _abi.load()
    odd = ctypes.c_void_p(0x1008)
    q = lambda rows=4, cols=64, br=1, dt=BF16, x=F: lib.cf_quantize_fp8(  # noqa: E731
        x, dt, F, F, rows, cols, br, None)
    assert q(rows=-1) == _abi.CF_ERR_INVALID_ARGUMENT
    assert q(x=None) == _abi.CF_ERR_INVALID_ARGUMENT
    assert q(rows=1 << 40, cols=1 << 20) == _abi.CF_ERR_INVALID_ARGUMENT
    assert q(br=2) == _abi.CF_ERR_UNSUPPORTED
    assert q(dt=7) == _abi.CF_ERR_UNSUPPORTED
    assert q(rows=0) == _abi.CF_OK and q(cols=0) == _abi.CF_OK
    mm = lambda m=4, k=64, n=64, dt=BF16, a=F, y=F, sc=F, pitch=None: (  # noqa: E731
        lib.cf_matmul_fp8(a, sc, m + -m % 4 if pitch is None else pitch, F, F, y, m, k, n, dt,
                          None))
    assert mm(m=-1) == _abi.CF_ERR_INVALID_ARGUMENT
    assert mm(a=None) == _abi.CF_ERR_INVALID_ARGUMENT
    assert mm(m=1 << 31) == _abi.CF_ERR_INVALID_ARGUMENT
    assert mm(m=1 << 30, n=1 << 30) == _abi.CF_ERR_INVALID_ARGUMENT
    assert mm(dt=F32) == _abi.CF_ERR_UNSUPPORTED
    assert mm(k=72) == _abi.CF_ERR_UNSUPPORTED and mm(k=0) == _abi.CF_ERR_UNSUPPORTED
    assert mm(a=odd) == _abi.CF_ERR_MISALIGNED and mm(y=odd) == _abi.CF_ERR_MISALIGNED
    assert mm(sc=odd) == _abi.CF_ERR_MISALIGNED
    assert mm(pitch=3) == _abi.CF_ERR_INVALID_ARGUMENT
    assert mm(pitch=6) == _abi.CF_ERR_UNSUPPORTED
    assert mm(m=0) == _abi.CF_OK and mm(n=0) == _abi.CF_OK
    lin = lambda m=40, k=64, x=F, ws=F, size=1 << 20: lib.cf_linear_fp8(  # noqa: E731
        x, F, F, F, m, k, 64, F16, ws, size, None)
    need = lib.cf_linear_fp8_workspace_bytes(40, 64)
    assert need == 40 * 64 + 40 * 4 and lib.cf_linear_fp8_workspace_bytes(0, 64) == 0
    assert lin(size=need - 1) == _abi.CF_ERR_WORKSPACE
    assert lin(ws=None) == _abi.CF_ERR_WORKSPACE
    assert lin(ws=odd) == _abi.CF_ERR_MISALIGNED and lin(x=odd) == _abi.CF_ERR_MISALIGNED
    assert lin(k=24) == _abi.CF_ERR_UNSUPPORTED
    assert lin(m=0) == _abi.CF_OK


def test_gated_linear_refuses():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.zeros(32, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="activation must be one of"):
        cf.gated_linear(x, w, w, "relu")
    with pytest.raises(ValueError, match="w_gate and w_up must both be"):
        cf.gated_linear(x, w, w[:16])
    with pytest.raises(ValueError, match="input features"):
        cf.gated_linear(x[:, :32], w, w)
    with pytest.raises(ValueError, match="one dtype"):
        cf.gated_linear(x, w, w.half())
    with pytest.raises(ValueError, match="one dtype"):
        cf.gated_linear(x.float(), w.float(), w.float())
    with pytest.raises(RuntimeError, match="CUDA"):
        cf.gated_linear(x, w, w)


def test_gated_linear_entry_points_refuse():
    lib = _abi.load()
    odd = ctypes.c_void_p(0x1008)

    def fwd(m=4, k=64, n=32, act=0, dt=BF16, x=F, g=None, u=None):
        return lib.cf_gated_linear(x, F, F, F, g, u, m, k, n, act, dt, None)

    assert fwd(m=-1) == _abi.CF_ERR_INVALID_ARGUMENT
    assert fwd(x=None) == _abi.CF_ERR_INVALID_ARGUMENT
    assert fwd(act=2) == _abi.CF_ERR_INVALID_ARGUMENT
    assert fwd(g=F) == _abi.CF_ERR_INVALID_ARGUMENT
    assert fwd(m=1 << 31) == _abi.CF_ERR_INVALID_ARGUMENT
    assert fwd(m=1 << 30, n=1 << 30) == _abi.CF_ERR_INVALID_ARGUMENT
    assert fwd(dt=F32) == _abi.CF_ERR_UNSUPPORTED
    assert fwd(k=60) == _abi.CF_ERR_UNSUPPORTED and fwd(n=36) == _abi.CF_ERR_UNSUPPORTED
    assert fwd(k=0) == _abi.CF_ERR_UNSUPPORTED
    assert fwd(x=odd) == _abi.CF_ERR_MISALIGNED and fwd(g=odd, u=F) == _abi.CF_ERR_MISALIGNED
    assert fwd(m=0) == _abi.CF_OK and fwd(n=0) == _abi.CF_OK
    need = lib.cf_gated_linear_backward_workspace_bytes(4, 32)
    assert need == 512 and lib.cf_gated_linear_backward_workspace_bytes(0, 32) == 0

    def bwd(m=4, g=F, dx=F, ws=F, size=need):
        return lib.cf_gated_linear_backward(F, F, F, F, g, F, dx, F, F, m, 64, 32, 1, F16, ws, size,
                                            None)

    assert bwd(g=None) == _abi.CF_ERR_INVALID_ARGUMENT
    assert bwd(ws=None) == _abi.CF_ERR_WORKSPACE and bwd(size=need - 1) == _abi.CF_ERR_WORKSPACE
    assert bwd(dx=odd) == _abi.CF_ERR_MISALIGNED and bwd(ws=odd) == _abi.CF_ERR_MISALIGNED
    assert bwd(m=0) == _abi.CF_OK
