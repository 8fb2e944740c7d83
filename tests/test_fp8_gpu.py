"""8-bit floating-point quantisation and products (quantize_fp8, matmul_fp8, linear_fp8).

A scale is one fp32 product with the fp32 number next to 1 / 448, a code one fp32 division and one
rounding, so they are compared bit for bit with torch's. Products are compared with 64-bit products of the dequantised operands: a
block's 128 products are exact and at most 36 additions deep on the tensor core, each off by at
most 2^-23 of the block's sum of |products|, and the blocks' sums add 2^-24 each, so with up to
2^6 blocks the fp32 value is within 2^-17 of the sum of |products|; rounding it adds half a step
of the result's type (and half of float16's smallest subnormal).
"""

from __future__ import annotations

import pytest
import torch

import cuda_force_b200 as cf

pytestmark = pytest.mark.gpu

BLOCK = 128


def reference_quantize(x, block_rows):
    rows, cols = x.shape
    rb, cb = -(-rows // block_rows), -(-cols // BLOCK)
    wide = torch.zeros(rb * block_rows, cb * BLOCK, device=x.device)
    wide[:rows, :cols] = x.float()
    blocks = wide.view(rb, block_rows, cb, BLOCK)
    top = blocks.abs().amax((1, 3))
    scales = top * (torch.ones((), device=x.device) / torch.full((), 448.0, device=x.device))
    scales = torch.where(scales > 0, scales, torch.ones_like(scales))
    codes = (blocks / scales[:, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.view(rb * block_rows, cb * BLOCK)[:rows, :cols].contiguous(), scales


def spread(scales, block_rows, rows, cols):
    return scales.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(
        BLOCK, 1)[:, :cols]


def assert_same(got, want, what):
    # NaN equals NaN whatever its bits.
    a, b = got.float(), want.float()
    assert torch.equal(a.isnan(), b.isnan()), what
    assert torch.equal(a.nan_to_num(0), b.nan_to_num(0)), what


def check_product(y, a, sa, w, sw):
    m, k = a.shape
    n = w.shape[0]
    a64 = a.double() * spread(sa, 1, m, k)
    w64 = w.double() * spread(sw, 128, n, k)
    ref = a64 @ w64.t()
    mag = a64.abs() @ w64.abs().t()
    tol = torch.finfo(y.dtype).eps / 2 * ref.abs() + 2.0**-17 * mag
    if y.dtype == torch.float16:
        tol = tol + 2.0**-25
    assert y.shape == (m, n)
    worst = ((y.double() - ref).abs() - tol).max().item()
    assert worst <= 0, f"{worst:.3g} over the bar"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 127), (130, 136), (128, 4096), (257, 1000),
                                   (300, 1029), (1000, 11008)])
def test_quantize_is_exact(shape, block_rows, dtype, cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(shape[0] * 7 + shape[1])
    x = torch.randn(shape, generator=g, device=cuda_device)
    x = torch.where(torch.rand(shape, generator=g, device=cuda_device) < 1e-3, 30 * x, x).to(dtype)
    codes, scales = cf.quantize_fp8(x, block_rows)
    ref_codes, ref_scales = reference_quantize(x, block_rows)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape
    assert scales.shape == ref_scales.shape and torch.equal(scales, ref_scales)
    assert torch.equal(codes.view(torch.uint8), ref_codes.view(torch.uint8))


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_special_blocks(block_rows, cuda_device):
    # One kind of block each: zeros, subnormals whose scale underflows or is tiny, huge values,
    # infinity, NaN, halfway points of the code grid, the smallest codes.
    x = torch.randn(block_rows, 10 * BLOCK, device=cuda_device)
    part = lambda i: x[:, i * BLOCK:(i + 1) * BLOCK]  # noqa: E731
    part(0).zero_()
    part(1).mul_(2.0**-149)
    part(2).mul_(2.0**-125)
    part(3).mul_(2.0**-60)
    part(4).mul_(2.0**124)
    part(5)[0, 3] = float("inf")
    part(6)[0, 5] = float("nan")
    part(6)[0, 6] = float("-inf")
    part(6)[0, 7] = 1e6
    # scale 1 exactly: values on and beside the midpoints of e4m3 neighbours
    grid = torch.arange(0, 127, dtype=torch.uint8, device=cuda_device).view(
        torch.float8_e4m3fn).float()
    mid = (grid[:-1] + grid[1:]) / 2
    part(7).zero_()
    part(7)[0, :126] = mid
    part(7)[0, 126:] = 448.0
    part(8)[0, :126] = torch.nextafter(mid, torch.zeros_like(mid))
    part(8)[0, 126:] = -448.0
    part(8)[1:].zero_()
    part(9)[0, :126] = -torch.nextafter(mid, torch.full_like(mid, 1e9))
    part(9)[0, 126:] = 448.0
    part(9)[1:].zero_()
    codes, scales = cf.quantize_fp8(x, block_rows)
    ref_codes, ref_scales = reference_quantize(x, block_rows)
    assert torch.equal(scales, ref_scales)
    assert_same(codes, ref_codes, "codes")
    assert scales[0, 0] == 1 and scales[0, 6] == 1 and scales[0, 7] == 1


def test_quantize_quotients_are_rounded_once(cuda_device):
    # The codes come without a division: every bf16 magnitude against scales of many mantissas.
    values = torch.arange(0x3000, 0x4380, dtype=torch.int16, device=cuda_device).view(torch.bfloat16)
    values = values.float()
    for top in (1.0, 448.0, 5.123, 3.0e-5, 77777.0, 0.999999):
        x = values[values <= top].view(-1)
        x = x[: x.numel() // 127 * 127].view(-1, 127)
        x = torch.cat([x, torch.full((x.shape[0], 1), top, device=cuda_device)], 1)
        codes, scales = cf.quantize_fp8(x)
        ref_codes, ref_scales = reference_quantize(x, 1)
        assert torch.equal(scales, ref_scales)
        assert torch.equal(codes.view(torch.uint8), ref_codes.view(torch.uint8))


def test_quantize_layouts(cuda_device):
    base = torch.randn(64, 7, 300, device=cuda_device, dtype=torch.bfloat16)
    x = base.transpose(0, 1)
    codes, scales = cf.quantize_fp8(x)
    assert codes.shape == x.shape and scales.shape == (7, 64, 3)
    ref_codes, ref_scales = reference_quantize(x.reshape(-1, 300), 1)
    assert torch.equal(codes.reshape(-1, 300).view(torch.uint8), ref_codes.view(torch.uint8))
    assert torch.equal(scales.reshape(-1, 3), ref_scales)
    off = torch.randn(4 * 256 + 1, device=cuda_device)[1:].view(4, 256)  # off the 16-byte boundary
    codes, scales = cf.quantize_fp8(off)
    assert torch.equal(codes.view(torch.uint8), reference_quantize(off, 1)[0].view(torch.uint8))
    for shape in ((0, 128), (5, 0)):
        codes, scales = cf.quantize_fp8(torch.zeros(shape, device=cuda_device))
        assert codes.shape == shape and scales.numel() == 0


SHAPES = [
    # (m, k, n): fused rows, streamed rows and tiles, at and around their limits
    (1, 128, 128), (1, 4096, 4096), (3, 16, 8), (8, 2000, 1030), (8, 8192, 700), (5, 1040, 5000),
    (9, 256, 264), (16, 4096, 4800), (17, 4160, 1030), (32, 1024, 11008), (31, 144, 33),
    (33, 128, 256), (64, 400, 300), (129, 4096, 256), (777, 4160, 1030), (256, 16, 512),
    (1000, 1152, 2051), (4096, 512, 4096), (300, 8192, 384),
    # few tiles: clusters of 2, 4 and 8 CTAs share a tile's k, ragged shares, odd features
    (40, 11008, 4096), (20, 1040, 2000), (100, 2064, 1031), (130, 4096, 200), (64, 8192, 64),
    (9, 4112, 7), (300, 1040, 129),
    # streamed: one feature, tiles of two sizes, several to a CTA, more than 32 stages a tile
    (1, 48, 1), (4, 144, 9), (6, 1024, 301), (7, 4224, 11008), (2, 33040, 600), (8, 32896, 2405),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_products(shape, dtype, cuda_device):
    m, k, n = shape
    g = torch.Generator(device=cuda_device).manual_seed(m + k + n)
    x = torch.randn(m, k, generator=g, device=cuda_device).to(dtype)
    x[:, : k // 2] *= 8  # blocks of unlike scales
    w = torch.randn(n, k, generator=g, device=cuda_device) * 0.02
    w[: n // 2] *= 5
    wc, ws = cf.quantize_fp8(w, 128)
    xc, xs = cf.quantize_fp8(x)
    y = cf.matmul_fp8(xc, xs, wc, ws, dtype)
    assert y.dtype == dtype
    check_product(y, xc, xs, wc, ws)
    # the linear is the same product of the same codes
    y2 = cf.linear_fp8(x, wc, ws)
    check_product(y2, xc, xs, wc, ws)
    assert torch.equal(cf.linear_fp8(x, wc, ws), y2)


@pytest.mark.parametrize("m", [1, 20, 200])
@pytest.mark.parametrize("k", [1, 100, 130, 1000])
def test_odd_feature_counts_are_padded(m, k, cuda_device):
    x = torch.randn(m, k, device=cuda_device).bfloat16()
    wc, ws = cf.quantize_fp8(torch.randn(77, k, device=cuda_device), 128)
    xc, xs = cf.quantize_fp8(x)
    check_product(cf.linear_fp8(x, wc, ws), xc, xs, wc, ws)


@pytest.mark.parametrize("m", [4, 24, 150])
def test_special_values_stay_where_they_are(m, cuda_device):
    x = torch.randn(m, 512, device=cuda_device).bfloat16()
    wc, ws = cf.quantize_fp8(torch.randn(300, 512, device=cuda_device), 128)
    clean = cf.linear_fp8(x, wc, ws)
    x[1, 200] = float("nan")
    x[3, 7] = float("inf")
    x[2] = 0
    y = cf.linear_fp8(x, wc, ws)
    assert y[1].isnan().all() and y[3].isnan().all() and torch.count_nonzero(y[2]) == 0
    keep = [i for i in range(m) if i not in (1, 2, 3)]
    assert torch.equal(y[keep], clean[keep])


def test_leading_dimensions_slices_and_empties(cuda_device):
    wc, ws = cf.quantize_fp8(torch.randn(96, 256, device=cuda_device), 128)
    x = torch.randn(2, 3, 256, device=cuda_device).bfloat16()
    y = cf.linear_fp8(x, wc, ws)
    assert y.shape == (2, 3, 96)
    assert torch.equal(y.view(6, 96), cf.linear_fp8(x.view(6, 256), wc, ws))
    # a slice that begins off the 16-byte boundary, and a transposed weight view
    buf = torch.randn(40 * 256 + 1, device=cuda_device).bfloat16()
    odd = buf[1:].view(40, 256)
    assert torch.equal(cf.linear_fp8(odd, wc, ws), cf.linear_fp8(odd.clone(), wc, ws))
    assert cf.linear_fp8(x[:0], wc, ws).shape == (0, 3, 96)
    assert cf.linear_fp8(x, wc[:0], ws[:0]).shape == (2, 3, 0)
    none = torch.empty(4, 0, device=cuda_device).bfloat16()
    zero = cf.linear_fp8(none, *cf.quantize_fp8(torch.empty(9, 0, device=cuda_device), 128))
    assert zero.shape == (4, 9) and torch.count_nonzero(zero) == 0


def test_rows_behind_the_last_are_left_alone(cuda_device):
    # Through the C entry: an output buffer longer than m rows.
    from cuda_force_b200 import _abi
    from tests.helpers import ptr, stream_ptr

    lib = _abi.load()
    for m in (3, 20, 130):
        x = torch.randn(m, 256, device=cuda_device).bfloat16()
        wc, ws = cf.quantize_fp8(torch.randn(200, 256, device=cuda_device), 128)
        y = torch.full((m + 130, 200), 7.0, device=cuda_device).bfloat16()
        need = lib.cf_linear_fp8_workspace_bytes(m, 256)
        work = torch.empty(max(need, 16), dtype=torch.uint8, device=cuda_device)
        assert lib.cf_linear_fp8(ptr(x), ptr(wc), ptr(ws), ptr(y), m, 256, 200, _abi.CF_DTYPE_BF16,
                                 ptr(work), need, stream_ptr()) == _abi.CF_OK
        torch.cuda.synchronize()
        assert (y[m:] == 7).all()
        assert torch.equal(y[:m], cf.linear_fp8(x, wc, ws))
        if need:
            assert lib.cf_linear_fp8(ptr(x), ptr(wc), ptr(ws), ptr(y), m, 256, 200,
                                     _abi.CF_DTYPE_BF16, ptr(work), need - 1,
                                     stream_ptr()) == _abi.CF_ERR_WORKSPACE


def test_side_stream_and_graphs(cuda_device):
    wc, ws = cf.quantize_fp8(torch.randn(640, 512, device=cuda_device), 128)
    xs = [torch.randn(m, 512, device=cuda_device).bfloat16() for m in (4, 40, 300)]
    eager = [cf.linear_fp8(x, wc, ws) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = [cf.linear_fp8(x, wc, ws) for x in xs]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, on_side))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [cf.linear_fp8(x, wc, ws) for x in xs]
        graphs.append((graph, out))
    xs[1].mul_(0.5)
    eager = [cf.linear_fp8(x, wc, ws) for x in xs]
    for graph, out in (graphs[1], graphs[0], graphs[1]):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, out))


def test_device_status_is_clean(cuda_device):
    from cuda_force_b200 import _abi

    assert _abi.load().cf_device_status() == _abi.CF_OK
