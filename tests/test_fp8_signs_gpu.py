"""The signs of quantised zeros (quantize_fp8): code = e4m3(fl32(x / scale)) for -0.0 too."""

from __future__ import annotations

import pytest
import torch

import cuda_force_b200 as cf

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("cols", [512, 130])  # whole accesses, element by element
def test_zeros_keep_their_signs(cols, block_rows, dtype, cuda_device):
    # Zeros of both signs, and values small enough that their codes are zeros, in blocks of
    # ordinary magnitude, of all zeros, and (in float32) of the smallest and largest scales.
    g = torch.Generator(device=cuda_device).manual_seed(cols)
    rows = 5 * 128
    top = torch.ones(rows, 1, device=cuda_device)
    top[128:256] = 0
    if dtype == torch.float32:
        top[256:384] = 2.0**-120
        top[384:512] = 2.0**120
    top[512:] = 2.0**-10
    x = torch.randn(rows, cols, generator=g, device=cuda_device) * top
    kind = torch.randint(4, x.shape, generator=g, device=cuda_device)
    x = torch.where(kind == 0, 0.0, x)
    x = torch.where(kind == 1, -0.0, x)
    x = torch.where(kind == 2, x * 2.0**-14, x).to(dtype)
    codes, scales = cf.quantize_fp8(x, block_rows)
    spread = scales.repeat_interleave(block_rows, 0).repeat_interleave(128, 1)[:rows, :cols]
    want = (x.float() / spread).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    assert torch.equal(codes.view(torch.uint8), want)
    zeros = x == 0
    assert torch.equal(codes.view(torch.uint8)[zeros] == 0x80, x[zeros].signbit())
