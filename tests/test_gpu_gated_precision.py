"""What the gated scan holds in float32 is as exact as float32 sums make it, whatever the inputs' type.

A rounding of a sum to float32 is off by at most 2^-24 of it, 2^-24 / sqrt(3) = 3.4e-8 in the root mean square. A chunk's state
comes of four products after each other (the inverse, K H, T R, K^T Delta) of at most 64 terms each at widths up to 64 and 128
above, 256 to 384 roundings of random sign: sqrt(384) * 3.4e-8 = 6.7e-7 of the 2-norm, and chunks before it fade: 1e-6. The
gradients go through as many again behind the forward's: 2e-6. Operands of two bfloat16 pieces in place of three leave 4e-6 on
the states and 8e-6 on the decays' gradients.
"""

from __future__ import annotations

import pytest
import torch

from conftest import needs_gpu
from oracle.gated import gated_scan
from test_gpu_gated_scan import BF16, F32, GPU, _inputs

pytestmark = [pytest.mark.gpu, needs_gpu]


def _off(got, want):
    got = got.detach().cpu().double()
    return float((got - want.detach()).norm() / want.detach().norm())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [(2, 300, 4, 64), (2, 250, 2, 128), (3, 150, 3, 16), (1, 200, 2, 200), (1, 2100, 2, 64)], ids=str)
def test_states_and_float32_gradients(dtype, size):
    from vesper.kernels.gated_scan import gated_delta_scan

    b, n, h, dk = size
    inputs = _inputs(*size, dtype, seed=sum(size) + 2)
    gen = torch.Generator().manual_seed(5)
    do, ds = torch.randn(b, n, h, dk, generator=gen).to(GPU, dtype), torch.randn(b, h, dk, dk, generator=gen).to(GPU)
    leaves = [t.requires_grad_() for t in inputs]
    o, after = gated_delta_scan(*leaves)
    dg, dstate = torch.autograd.grad([o, after], leaves[4:], [do, ds])
    exact = [t.detach().cpu().double().requires_grad_() for t in inputs]
    want_o, want_after = gated_scan(*exact)
    want_dg, want_dstate = torch.autograd.grad([want_o, want_after], exact[4:], [do.cpu().double(), ds.cpu().double()])
    offs = {"state": _off(after, want_after), "dg": _off(dg, want_dg), "dstate": _off(dstate, want_dstate)}
    assert offs["state"] <= 1e-6 and offs["dg"] <= 2e-6 and offs["dstate"] <= 2e-6, offs
