"""The oracle of the gated delta rule and the layer norm: closed forms, invariants, gradients by differences; and the
plain chunked scan of ``vesper.recurrence`` against it."""

from __future__ import annotations

import math

import pytest
import torch

from oracle.delta import delta_scan_step
from oracle.gated import gated_scan, gated_step, layer_norm

F64 = torch.float64


def _inputs(b, n, h, dk, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(b, n, h, dk, generator=g, dtype=F64) for _ in range(3))
    k = k / k.norm(dim=-1, keepdim=True)
    beta = torch.rand(b, n, h, generator=g, dtype=F64)
    decay = -torch.rand(b, n, h, generator=g, dtype=F64)
    return q, k, v, beta, decay, torch.randn(b, h, dk, dk, generator=g, dtype=F64)


def test_one_token_of_one_feature_by_hand():
    one = lambda x: torch.tensor([[[x]]], dtype=F64)  # noqa: E731
    gate = lambda x: torch.tensor([[x]], dtype=F64)  # noqa: E731
    o, after = gated_step(one(2.0), one(1.0), one(3.0), gate(0.5), gate(math.log(0.25)), torch.full((1, 1, 1, 1), 8.0, dtype=F64))
    # faded 8 / 4 = 2, correction 0.5 (3 - 2) = 0.5, state 2.5, read 5
    assert torch.allclose(after, torch.full_like(after, 2.5)) and torch.allclose(o, torch.full_like(o, 5.0))


def test_without_decay_it_is_the_delta_rule():
    q, k, v, beta, _, state = _inputs(2, 1, 3, 5)
    mine = gated_step(q[:, 0], k[:, 0], v[:, 0], beta[:, 0], torch.zeros_like(beta[:, 0]), state)
    theirs = delta_scan_step(q[:, 0], k[:, 0], v[:, 0], beta[:, 0], state)
    for a, b in zip(mine, theirs):
        assert torch.allclose(a, b, rtol=1e-13, atol=1e-13)


def test_a_decay_of_minus_infinity_starts_anew():
    q, k, v, beta, g, state = _inputs(1, 6, 2, 4)
    g[:, 3] = -math.inf
    whole, after = gated_scan(q, k, v, beta, g, state)
    fresh, alone = gated_scan(*(t[:, 3:] for t in (q, k, v, beta, g)), torch.zeros_like(state))
    assert torch.equal(whole[:, 3:], fresh) and torch.equal(after, alone)


def test_gradients_by_differences():
    inputs = [t.requires_grad_() for t in _inputs(1, 3, 1, 2)]
    assert torch.autograd.gradcheck(lambda *a: gated_scan(*a), inputs)
    x, r = (torch.randn(3, 4, dtype=F64, requires_grad=True) for _ in range(2))
    gain, bias = (torch.randn(4, dtype=F64, requires_grad=True) for _ in range(2))
    assert torch.autograd.gradcheck(lambda *a: layer_norm(*a, 1e-5), (x, gain, bias, r))


def test_layer_norm_of_two_values_by_hand():
    x = torch.tensor([[1.0, 5.0]], dtype=F64)
    y, s = layer_norm(x, torch.tensor([1.0, 2.0], dtype=F64), torch.tensor([0.5, 0.0], dtype=F64), torch.ones_like(x), 0.0)
    assert torch.equal(s, x + 1) and torch.allclose(y, torch.tensor([[-0.5, 2.0]], dtype=F64))


@pytest.mark.parametrize("n", [0, 1, 5, 64, 130])
@pytest.mark.parametrize("block", [1, 16, 64])
def test_the_plain_chunked_scan_is_the_oracle(n, block):
    from vesper.recurrence import gated_delta_scan_chunked

    q, k, v, beta, g, state = _inputs(2, n, 3, 8, seed=n)
    if n > 3:
        g[0, 3] = -math.inf
    active = torch.arange(2 * n).view(2, n) % 3 != 0
    o, after = gated_delta_scan_chunked(q, k, v, beta, g, state, block, active=active)
    want, last = gated_scan(q, k, v, beta, g, state, active)
    assert torch.allclose(o, want, rtol=1e-9, atol=1e-11) and torch.allclose(after, last, rtol=1e-9, atol=1e-11)
    if n == 0:
        assert o is q and after is state


def test_the_plain_chunked_scan_s_gradients():
    from vesper.recurrence import gated_delta_scan_chunked

    inputs = _inputs(1, 21, 2, 4, seed=3)
    grads = []
    for scan in (lambda *a: gated_delta_scan_chunked(*a, 8), gated_scan):
        leaves = [t.clone().requires_grad_() for t in inputs]
        o, after = scan(*leaves)
        grads.append(torch.autograd.grad(o.sin().sum() + after.cos().sum(), leaves))
    for a, b in zip(*grads):
        assert torch.allclose(a, b, rtol=1e-8, atol=1e-10)
