"""Empty batches through the gated scan and the layer norm: empty results that every input has a gradient from. On the
CPU: no kernel is reached."""

from __future__ import annotations

import pytest
import torch

from test_gated_refusals import _on

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _leaf(*shape, dtype=F32):
    return _on(torch.zeros(*shape, dtype=dtype)).requires_grad_()


@pytest.mark.parametrize("types", [(F32, F32, F32), (F32, BF16, F16), (BF16, BF16, BF16)], ids=str)
@pytest.mark.parametrize("lead", [(0,), (3, 0), (0, 2)], ids=str)
def test_the_norm_of_no_rows_has_every_gradient(types, lead):
    from vesper.kernels.layer_norm import layer_norm

    x, r = _leaf(*lead, 24, dtype=types[0]), _leaf(*lead, 24, dtype=types[1])
    gain, bias = _leaf(24), _leaf(24)
    y, s = layer_norm(x, gain, bias, residual=r, dtype=types[2])
    assert y.shape == s.shape == x.shape and y.dtype == types[2] and s.dtype == types[0]
    grads = torch.autograd.grad([y, s], [x, gain, bias, r], [torch.zeros_like(y), torch.zeros_like(s)])
    for leaf, grad in zip((x, gain, bias, r), grads):
        assert grad.shape == leaf.shape and grad.dtype == leaf.dtype and not bool(grad.any())
    y = layer_norm(x, gain, bias, dtype=types[2])  # without a residual
    assert not bool(torch.autograd.grad(y.sum(), bias)[0].any())
    only = layer_norm(x.detach(), gain.detach(), bias, dtype=types[2])  # the bias alone
    assert only.requires_grad and not bool(torch.autograd.grad(only.sum(), bias)[0].any())
    with torch.no_grad():
        assert not layer_norm(x, gain, bias, dtype=types[2]).requires_grad


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize(("b", "n", "h", "dk"), [(0, 5, 2, 16), (2, 5, 0, 16), (0, 1, 2, 12), (0, 3, 0, 1)])
def test_the_scan_of_an_empty_batch_has_every_gradient(dtype, b, n, h, dk):
    from vesper.kernels.gated_scan import gated_delta_scan

    leaves = [*(_leaf(b, n, h, dk, dtype=dtype) for _ in range(3)), _leaf(b, n, h, dtype=dtype), _leaf(b, n, h), _leaf(b, h, dk, dk)]
    o, after = gated_delta_scan(*leaves, active=_on(torch.ones(b, n, dtype=torch.bool)))
    assert o.shape == leaves[0].shape and o.dtype == dtype and after.shape == leaves[5].shape and after.dtype == F32
    for result in (o, after):
        grads = torch.autograd.grad(result.sum(), leaves, retain_graph=True)
        for leaf, grad in zip(leaves, grads):
            assert grad.shape == leaf.shape and grad.dtype == leaf.dtype
    only = gated_delta_scan(*(t.detach() for t in leaves[:4]), leaves[4], leaves[5].detach())  # the decays alone
    assert all(t.requires_grad for t in only)
    with torch.no_grad():
        o, after = gated_delta_scan(*leaves)
    assert not o.requires_grad and not after.requires_grad and after is not leaves[5]
