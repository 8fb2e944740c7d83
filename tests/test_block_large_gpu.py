"""The feed-forward block's operators on tensors of more than 2^31 elements: sampled rows at the
start, around element 2^31 and at the end against the formulas in 64 bits. Bars as in each
operator's own tests: half a step of the result's type and a few fp32 roundings (2^-18 of the sum
of |terms| covers the short sums here)."""

from __future__ import annotations

import pytest
import torch

import cuda_force_b200 as cf

pytestmark = pytest.mark.gpu

EDGE = 2**31


def sampled(rows, cols):
    edge = EDGE // cols
    return sorted({0, 1, edge - 1, edge, edge + 1, rows // 2 + 7, rows - 2, rows - 1})


def test_quantize(cuda_device):
    cols = 1544  # not a whole number of blocks
    rows = EDGE // cols + 300
    x = torch.empty(rows, cols, device=cuda_device, dtype=torch.bfloat16).normal_()
    inverse = torch.ones((), device=cuda_device) / torch.full((), 448.0, device=cuda_device)
    codes, scales = cf.quantize_fp8(x)
    for r in sampled(rows, cols):
        wide = torch.nn.functional.pad(x[r].float(), (0, -cols % 128)).view(-1, 128)
        want = wide.abs().amax(1) * inverse
        assert torch.equal(scales[r], want)
        c = (wide / want[:, None]).to(torch.float8_e4m3fn).view(-1)[:cols]
        assert torch.equal(codes[r].view(torch.uint8), c.view(torch.uint8))
    codes, scales = cf.quantize_fp8(x, block_rows=128)
    for r in sampled(rows, cols):
        top = r // 128 * 128
        wide = torch.nn.functional.pad(x[top:top + 128].float(), (0, -cols % 128))
        want = wide.abs().amax(0).view(-1, 128).amax(1) * inverse
        assert torch.equal(scales[r // 128], want)
        c = (wide[r - top] / want.repeat_interleave(128)).to(torch.float8_e4m3fn)[:cols]
        assert torch.equal(codes[r].view(torch.uint8), c.view(torch.uint8))


@pytest.mark.parametrize("cols", [2048, 2047])
def test_norm(cols, cuda_device):
    rows = EDGE // cols + 200
    x = torch.empty(rows, cols, device=cuda_device, dtype=torch.bfloat16).normal_()
    r = torch.empty_like(x).normal_()
    w = (1 + 0.1 * torch.randn(cols, device=cuda_device)).bfloat16()
    xs, rs = x.requires_grad_(), r.requires_grad_()
    n, h = cf.gated_residual_rmsnorm(xs, rs, w, w)
    dx, dr = torch.autograd.grad((n, h), (xs, rs), (x.detach(), r.detach()))
    at = sampled(rows, cols)
    x64 = x.detach()[at].double().requires_grad_()
    r64 = r.detach()[at].double().requires_grad_()
    norm = lambda v: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * w.double()  # noqa: E731
    h64 = r64 + norm(x64)
    n64 = norm(h64)
    want = torch.autograd.grad((n64, h64), (x64, r64), (x64.detach(), r64.detach()))
    for got, ref in ((n, n64), (h, h64), (dx, want[0]), (dr, want[1])):
        ref = ref.detach()
        tol = 2.0**-8 * ref.abs() + 2.0**-14 * ref.abs().max()
        assert ((got.detach()[at].double() - ref).abs() <= tol).all()


def test_linear_fp8(cuda_device):
    n, k = 2056, 128
    m = EDGE // n + 500
    x = torch.empty(m, k, device=cuda_device, dtype=torch.bfloat16).normal_()
    wc, ws = cf.quantize_fp8(torch.randn(n, k, device=cuda_device), 128)
    y = cf.linear_fp8(x, wc, ws)
    w64 = wc.double() * ws.double().repeat_interleave(128, 0)[:n]
    at = sampled(m, n)
    xc, xs = cf.quantize_fp8(x[at])
    x64 = xc.double() * xs.double()
    ref, mag = x64 @ w64.t(), x64.abs() @ w64.abs().t()
    assert ((y[at].double() - ref).abs() <= 2.0**-8 * ref.abs() + 2.0**-17 * mag).all()


def test_gated_linear(cuda_device):
    n, k = 2056, 64
    m = EDGE // n + 500
    x = torch.empty(m, k, device=cuda_device, dtype=torch.bfloat16).normal_().requires_grad_()
    wg, wu = ((torch.randn(n, k, device=cuda_device) * k**-0.5).bfloat16() for _ in range(2))
    y = cf.gated_linear(x, wg, wu)
    dy = torch.empty_like(y).normal_()
    (dx,) = torch.autograd.grad(y, x, dy)
    at = sampled(m, n)
    x64, g64, u64 = x.detach()[at].double(), wg.double(), wu.double()
    g, u = x64 @ g64.t(), x64 @ u64.t()
    s = torch.sigmoid(g)
    ref = g * s * u
    off = 2.0**-18 * ((x64.abs() @ g64.abs().t()) * u.abs() * 1.2
                      + (x64.abs() @ u64.abs().t()) * (g * s).abs() + 1)
    assert ((y.detach()[at].double() - ref).abs() <= 2.0**-8 * ref.abs() + off).all()
    d = dy[at].double()
    dg, du = d * u * (s + g * s * (1 - s)), d * g * s
    ref = dg @ g64 + du @ u64
    # dg and du are rounded once: 2^-8 of each, and another 2^-16 for their fp32 sums
    off = (2.0**-8 + 2.0**-16) * (dg.abs() @ g64.abs() + du.abs() @ u64.abs())
    assert ((dx[at].double() - ref).abs() <= 2.0**-8 * ref.abs() + off).all()
