"""The feed-forward block's operators as the dispatcher has them, without the Python wrappers, on
operands without input features: sums of nothing are zeros, in memory that held something else."""

from __future__ import annotations

import math

import pytest
import torch

import cuda_force_b200 as cf  # noqa: F401  registers the operators

pytestmark = pytest.mark.gpu


def spoil(device, *sizes):
    """Blocks of these many bytes that held NaN, free for the next allocations."""
    held = [torch.full((size // 2,), float("nan"), dtype=torch.bfloat16, device=device)
            for size in sizes]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("activation", [0, 1])
@pytest.mark.parametrize("lead", [(5,), (2, 3), (64,), ()], ids=str)
def test_gated_linear_without_input_features(lead, activation, cuda_device):
    n = 136
    op = torch.ops.cudaforge.gated_linear
    x = torch.empty(*lead, 0, dtype=torch.bfloat16, device=cuda_device)
    w = torch.empty(n, 0, dtype=torch.bfloat16, device=cuda_device)
    rows = math.prod(lead)
    for train in (False, True):
        leaves = [t.detach().clone().requires_grad_(train) for t in (x, w, w)]
        for _ in range(3):
            spoil(cuda_device, 2 * rows * n, 4 * rows * n, 4 * rows * n)
            y = op(*leaves, activation)
            assert y.shape == (*lead, n) and torch.count_nonzero(y) == 0
        if train:
            grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
            assert [g.shape for g in grads] == [t.shape for t in leaves]


@pytest.mark.parametrize("m", [0, 3, 40])
def test_products_without_input_features(m, cuda_device):
    x = torch.empty(m, 0, dtype=torch.bfloat16, device=cuda_device)
    wc, ws = torch.ops.cudaforge.quantize_fp8(torch.empty(70, 0, device=cuda_device), 128)
    xc, xs = torch.ops.cudaforge.quantize_fp8(x, 1)
    for _ in range(3):
        spoil(cuda_device, max(2, 2 * m * 70))
        y = torch.ops.cudaforge.linear_fp8(x, wc, ws)
        assert y.shape == (m, 70) and torch.count_nonzero(y) == 0
        spoil(cuda_device, max(2, 2 * m * 70))
        y = torch.ops.cudaforge.matmul_fp8(xc, xs, wc, ws, torch.bfloat16)
        assert y.shape == (m, 70) and torch.count_nonzero(y) == 0
