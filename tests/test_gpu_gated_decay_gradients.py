"""The log decays' gradients behind strong decays: small numbers beside the products they are made of.

Every term of a decay's gradient carries that decay, so that a sum of them is as exact as its terms: the bound of what is
held in float32, 6e-5 of the 2-norm (three sums of at most 320 terms after each other, 320 * 2^-24 = 1.9e-5 each), for each
head by itself and for the tokens of one decay by themselves. (As a difference of terms without it, in float32, the
gradient is off by 8e-5 at decays of e^-5, 7e-3 at e^-10 and a hundred times itself at e^-20.)
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import needs_gpu
from oracle.gated import gated_scan

pytestmark = [pytest.mark.gpu, needs_gpu]

GPU = torch.device("cuda")
BF16, F32 = torch.bfloat16, torch.float32
HELD32 = 6e-5


def _inputs(b, n, h, dk, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(b, n, h, dk, generator=gen) for _ in range(3))
    k = k / k.norm(dim=-1, keepdim=True)
    beta = torch.sigmoid(torch.randn(b, n, h, generator=gen))
    state = 0.5 * torch.randn(b, h, dk, dk, generator=gen)
    do, ds = torch.randn(b, n, h, dk, generator=gen), torch.randn(b, h, dk, dk, generator=gen)
    return [t.to(GPU, dtype) for t in (q, k, v, beta)], state.to(GPU), do.to(GPU, dtype), ds.to(GPU)


def _both(tokens, g, state, do, ds, active=None):
    """The decays' gradients of the kernels and of the float64 oracle."""
    from vesper.kernels.gated_scan import gated_delta_scan

    leaf = g.to(GPU).requires_grad_()
    o, after = gated_delta_scan(*tokens, leaf, state, active=active)
    got, = torch.autograd.grad([o, after], leaf, [do, ds])
    exact = g.double().requires_grad_()
    o, after = gated_scan(*(t.cpu().double() for t in tokens), exact, state.cpu().double(), None if active is None else active.cpu())
    want, = torch.autograd.grad([o, after], exact, [do.cpu().double(), ds.cpu().double()])
    return got.cpu().double(), want


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [(1, 140, 32), (2, 64, 8), (1, 65, 64), (1, 129, 72), (1, 100, 128), (1, 70, 256), (90, 130, 16)], ids=str)
def test_heads_of_one_decay_each(dtype, size):
    b, n, dk = size
    decays = torch.tensor([-1e-3, -1.0, -5.0, -10.0, -20.0, -50.0])
    tokens, state, do, ds = _inputs(b, n, 6, dk, dtype, seed=n + dk)
    got, want = _both(tokens, decays.expand(b, n, 6).clone(), state, do, ds)
    for head, decay in enumerate(decays):
        x, y = got[:, :, head], want[:, :, head]
        assert torch.isfinite(x).all()
        assert float((x - y).norm()) <= HELD32 * float(y.norm()), (float(decay), float((x - y).norm() / y.norm()))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dk", [16, 64])
def test_tokens_that_forget_much_among_tokens_that_keep(dtype, dk):
    gen = torch.Generator().manual_seed(dk)
    tokens, state, do, ds = _inputs(2, 150, 3, dk, dtype, seed=dk)
    kind = torch.randint(0, 4, (2, 150, 3), generator=gen)
    decays = torch.tensor([-0.01, -8.0, -16.0, -25.0])
    active = (torch.rand(2, 150, generator=gen) < 0.8).to(GPU)
    got, want = _both(tokens, decays[kind], state, do, ds, active)
    for i, decay in enumerate(decays):
        x, y = got[kind == i], want[kind == i]
        assert float((x - y).norm()) <= HELD32 * float(y.norm()), (float(decay), float((x - y).norm() / y.norm()))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decays_of_nothing_left_beside_slow_ones(dtype):
    """Sums of -19200 a chunk, in float64 before their differences: the gradients of the slow decays at the bound of the rest,
    those of e^-300 zeros."""
    tokens, state, do, ds = _inputs(1, 140, 2, 32, dtype, seed=11)
    g = torch.full((1, 140, 2), -300.0)
    g[:, ::3] = -1e-3
    got, want = _both(tokens, g, state, do, ds)
    assert float((got - want).norm()) <= HELD32 * float(want.norm())
    assert not bool(got[g < -1].any())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_forgetting_tokens_and_those_around_them(dtype):
    """-inf has a gradient of 0; the tokens of its chunk keep theirs."""
    tokens, state, do, ds = _inputs(1, 200, 2, 32, dtype, seed=3)
    g = -torch.rand(1, 200, 2, generator=torch.Generator().manual_seed(1)) * 6
    g[:, ::17] = -math.inf
    got, want = _both(tokens, g, state, do, ds)
    want = torch.nan_to_num(want)
    assert float((got - want).norm()) <= HELD32 * float(want.norm())
    assert not bool(got[torch.isinf(g)].any())
