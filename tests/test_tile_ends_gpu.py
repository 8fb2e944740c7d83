"""Tile kernels launched one after another with fewer 128-byte blocks of k than their rings have
stages, as many, and more: every launch gives the same bits, and no wait ran out."""

from __future__ import annotations

import pytest
import torch

import cuda_force_b200 as cf
from cuda_force_b200 import _abi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [64, 128, 384, 768, 1040])
def test_short_products_back_to_back(k, cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(k)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda_device).bfloat16()  # noqa: E731
    xs = [r(m, k) for m in (200, 2048)]
    wg, wu = r(2048, k), r(2048, k)
    wc, ws = cf.quantize_fp8(r(4096, k), 128)
    dys = [r(x.shape[0], 2048) for x in xs]
    for t in (*xs, wg, wu):
        t.requires_grad_()

    def once():
        out = []
        for x, dy in zip(xs, dys):
            out.append(cf.linear_fp8(x.detach(), wc, ws))
            y = cf.gated_linear(x, wg, wu)
            out += [y.detach(), *torch.autograd.grad(y, (x, wg, wu), dy)]
        return out

    first = once()
    for _ in range(30):
        again = once()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    assert _abi.load().cf_device_status() == _abi.CF_OK
