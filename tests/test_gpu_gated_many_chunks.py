"""The gated scan over more chunks than either form of its factors' kernels takes by lines (256 in bfloat16, 512 in
float32): against the oracle, and rows of a batch bit for bit as alone."""

from __future__ import annotations

import pytest
import torch

from conftest import needs_gpu
from test_gpu_gated_scan import BF16, F32, GPU, NAMES, _inputs, test_gradients_match_the_oracle as _gradients, \
    test_scan_matches_the_oracle as _scan

pytestmark = [pytest.mark.gpu, needs_gpu]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [(33, 130, 6, 16), (20, 70, 15, 32), (41, 200, 4, 64), (19, 65, 14, 128), (2, 5, 260, 136), (2, 3, 257, 256)], ids=str)
def test_scans_of_more_chunks_match_the_oracle(dtype, size):
    _scan(dtype, size, True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [(33, 130, 6, 16), (44, 150, 4, 64), (20, 65, 13, 72)], ids=str)
def test_gradients_of_more_chunks_match_the_oracle(dtype, size):
    _gradients(dtype, size, True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dk", [32, 64, 128, 256])
@pytest.mark.parametrize("b", [130, 180])  # 390 and 540 chunks: between the two types' limits, and past both
def test_a_row_among_more_is_the_row_alone(dtype, dk, b):
    from vesper.kernels.gated_scan import gated_delta_scan

    inputs = _inputs(b, 130, 1, dk, dtype, seed=dk, resets=True)
    do = torch.randn(b, 130, 1, dk, device=GPU, generator=torch.Generator(GPU).manual_seed(1)).to(dtype)
    leaves = [t.detach().requires_grad_() for t in inputs]
    o, after = gated_delta_scan(*leaves)
    grads = torch.autograd.grad([o, after], leaves, [do, torch.ones_like(after)])
    for row in (0, b // 2, b - 1):
        alone = [t[row : row + 1].detach().clone().requires_grad_() for t in inputs]
        o1, after1 = gated_delta_scan(*alone)
        grads1 = torch.autograd.grad([o1, after1], alone, [do[row : row + 1].clone(), torch.ones_like(after1)])
        for name, x, y in zip(("o", "state", *NAMES), (o, after, *grads), (o1, after1, *grads1)):
            assert torch.equal(x[row : row + 1], y), (name, row)
