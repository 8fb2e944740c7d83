"""The C entries of the feed-forward block's operators, called as the header allows and the
Python wrappers never do."""

from __future__ import annotations

import pytest
import torch

from cuda_force_b200 import _abi
from tests.helpers import TORCH_TO_CF, ptr, stream_ptr

pytestmark = pytest.mark.gpu


def norm_backward(x, residual, weight, post, gate, groups, dn, dh, stats):
    """The gradients of x, residual, weight, post_weight and gate by the C entry."""
    rows, cols = x.shape
    code = TORCH_TO_CF[x.dtype]
    null = lambda t: None if t is None else ptr(t)  # noqa: E731
    grads = [torch.empty_like(t) if t is not None else None
             for t in (x, residual, weight, post, gate)]
    lib = _abi.load()
    need = lib.cf_gated_residual_rmsnorm_backward_workspace_bytes(
        rows, cols, int(post is not None), 0 if gate is None else groups, code)
    work = torch.empty(need, dtype=torch.uint8, device=x.device)
    assert lib.cf_gated_residual_rmsnorm_backward(
        ptr(dn), ptr(dh), ptr(x), ptr(residual), ptr(weight), null(post), null(gate), groups,
        TORCH_TO_CF[weight.dtype], ptr(stats), *map(null, grads), rows, cols, 0.5, code, ptr(work),
        need, stream_ptr()) == _abi.CF_OK
    return [g for g in grads if g is not None]


def norm_inputs(rows, cols, dtype, device):
    g = torch.Generator(device=device).manual_seed(rows + cols)
    wide = [torch.randn(rows, cols, generator=g, device=device).to(dtype) for _ in range(4)]
    return wide, [torch.rand(cols, generator=g, device=device).to(dtype) for _ in range(3)]


def norm_forward(x, residual, weight, post, gate, groups, stats):
    n, h = torch.empty_like(x), torch.empty_like(x)
    code = TORCH_TO_CF[x.dtype]
    assert _abi.load().cf_gated_residual_rmsnorm(
        ptr(x), ptr(residual), ptr(weight), None if post is None else ptr(post),
        None if gate is None else ptr(gate), groups, TORCH_TO_CF[weight.dtype], ptr(n), ptr(h),
        ptr(stats), *x.shape, 0.5, 1e-6, code, stream_ptr()) == _abi.CF_OK
    return n, h


@pytest.mark.parametrize("shape, dtype", [
    ((7, 256), torch.bfloat16),     # a row for each warp
    ((300, 4096), torch.float16),   # rows that fill their threads' registers
    ((5, 1000), torch.float32),
    ((6, 333), torch.float32),      # element by element
    ((3, 9000), torch.bfloat16),    # long rows
], ids=str)
def test_norm_statistics_on_a_four_byte_boundary(shape, dtype, cuda_device):
    # stats is a float pointer: wherever a float may lie, the results are the same bits.
    rows, cols = shape
    (x, residual, dn, dh), (weight, post, gate) = norm_inputs(rows, cols, dtype, cuda_device)
    results = []
    for offset in (0, 1):
        stats = torch.full((2 * rows + 2,), float("nan"), device=cuda_device)[offset:]
        assert stats.data_ptr() % 8 == 4 * offset
        out = norm_forward(x, residual, weight, post, gate, 1, stats)
        assert not stats[:2 * rows].isnan().any() and stats[2 * rows:].isnan().all()
        results.append([*out, *norm_backward(x, residual, weight, post, gate, 1, dn, dh, stats)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("rows, cols", [(7, 256), (6, 333), (3, 9000)])
def test_norm_without_a_gate_has_no_gate_groups(rows, cols, cuda_device):
    # 0, which the workspace's size takes for no gate, and any other number.
    (x, residual, dn, dh), (weight, post, _) = norm_inputs(rows, cols, torch.float32, cuda_device)
    results = []
    for groups in (1, 0, -1, 5):
        stats = torch.empty(rows, 2, device=cuda_device)
        out = norm_forward(x, residual, weight, post, None, groups, stats)
        results.append([*out, *norm_backward(x, residual, weight, post, None, groups, dn, dh,
                                             stats)])
    torch.cuda.synchronize()
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
