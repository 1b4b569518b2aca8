"""The gated step of more heads than one launch takes, and a scan of one token that runs as it."""

from __future__ import annotations

import pytest
import torch

from conftest import needs_gpu
from oracle.gated import gated_step

pytestmark = [pytest.mark.gpu, needs_gpu]

GPU = torch.device("cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_heads_than_a_launch(dtype):
    from vesper.kernels.gated_scan import gated_delta_scan, gated_delta_step

    b, h, dk = 2**16 + 5, 16, 8
    gen = torch.Generator(device=GPU).manual_seed(0)
    q, k, v = (torch.randn(b, h, dk, device=GPU, generator=gen).to(dtype) for _ in range(3))
    beta = torch.rand(b, h, device=GPU, generator=gen).to(dtype)
    g, state = -torch.rand(b, h, device=GPU, generator=gen), torch.randn(b, h, dk, dk, device=GPU, generator=gen)
    k = k * 0.3
    active = torch.arange(b, device=GPU) % 3 != 1
    tokens = (q, k, v, beta, g)
    with torch.no_grad():
        o, after = gated_delta_scan(*(t[:, None] for t in tokens), state, active=active[:, None])
        whole, new = gated_delta_step(*tokens, state, active=active)
        assert torch.equal(o[:, 0], whole) and torch.equal(after, new)
        for start in (0, b // 2, b - 9):  # rows by themselves, in one launch
            rows = slice(start, start + 9)
            alone, last = gated_delta_step(*(t[rows] for t in tokens), state[rows].contiguous(), active=active[rows])
            assert torch.equal(whole[rows], alone) and torch.equal(new[rows], last)
            want, exact = gated_step(*(t[rows].cpu().double() for t in (*tokens, state)))
            want = want * active[rows].cpu()[:, None, None]
            # held in dtype: half a step of each value; sums of 8 products and three roundings in float32
            assert float((alone.cpu().double() - want).norm()) <= (torch.finfo(dtype).eps / 2 + 2e-6) * float(want.norm())
            assert float((last.cpu().double() - exact).norm()) <= 2e-6 * float(exact.norm())
        inplace = state.clone()
        again, same = gated_delta_step(*tokens, inplace, active=active, out_state=inplace)
        assert same is inplace and torch.equal(inplace, new) and torch.equal(again, whole)
