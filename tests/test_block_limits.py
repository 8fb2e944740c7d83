"""Sizes that the feed-forward block's C entries refuse before any CUDA call."""

from __future__ import annotations

import ctypes

from cuda_force_b200 import _abi

P = ctypes.c_void_p(0x1000)


def test_linear_fp8_takes_no_longer_rows_than_its_quantiser():
    # The quantiser's offsets inside a CTA are 32-bit: rows of up to 2^30 elements.
    lib = _abi.load()
    for k in ((1 << 30) + 16, (1 << 31) - 4096):
        assert lib.cf_quantize_fp8(P, _abi.CF_DTYPE_BF16, P, P, 2, k, 1, None) == (
            _abi.CF_ERR_INVALID_ARGUMENT)
        assert lib.cf_linear_fp8(P, P, P, P, 2, k, 64, _abi.CF_DTYPE_BF16, P, 1 << 62, None) == (
            _abi.CF_ERR_INVALID_ARGUMENT)
    assert lib.cf_linear_fp8(P, P, P, P, 2, 1 << 30, 64, _abi.CF_DTYPE_BF16, P, 0, None) == (
        _abi.CF_ERR_WORKSPACE)
