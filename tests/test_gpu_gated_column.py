"""A recurrent sublayer that normalizes its input and forgets: layer norm, projections, key filter, gated scan and output
projection as they run together in training and decoding."""

from __future__ import annotations

import pytest
import torch

from conftest import needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]

GPU = torch.device("cuda")


def _layer(seed=3, d=128, heads=2):
    from vesper.column import RecurrentSublayer

    gen = torch.Generator().manual_seed(seed)
    layer = RecurrentSublayer(d, heads, key_conv=4, generator=gen, decay=True, norm=True)
    with torch.no_grad():
        layer.norm_gain.copy_(torch.exp(0.2 * torch.randn(d, generator=gen)))
        layer.norm_bias.copy_(0.1 * torch.randn(d, generator=gen))
    dk = d // heads
    x = 2 * torch.randn(2, 150, d, generator=gen) + 1
    state, history = 0.1 * torch.randn(2, heads, dk, dk, generator=gen), torch.randn(2, 3, d, generator=gen)
    return layer.to(GPU), x.to(GPU), state.to(GPU), history.to(GPU)


def _off(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize(("impl", "bound"), [("fused-fp32", 1e-5), ("fused", 1.5e-2)])
def test_the_hip_scans_and_norm_against_plain_pytorch(impl, bound):
    """Outputs at the scan switch's bounds; gradients, which pass the projections' sums again, at four times them."""
    from vesper.column import set_scan

    layer, x, state, history = _layer()
    gen = torch.Generator().manual_seed(1)
    dy, ds = torch.randn(x.shape, generator=gen).to(GPU), torch.randn(state.shape, generator=gen).to(GPU)
    results = []
    for chosen in ("reference", impl):
        set_scan(layer, chosen)
        leaves = [x.detach().requires_grad_(), state.detach().requires_grad_(), *layer.parameters()]
        y, after, _ = layer(leaves[0], leaves[1], history)
        results.append([y, after, *torch.autograd.grad([y, after], leaves, [dy, ds])])
    names = ["y", "after", "x", "state", *(n for n, _ in layer.named_parameters())]
    assert {"w_decay", "decay_rate", "norm_gain", "norm_bias"} < set(names)
    for i, (name, a, b) in enumerate(zip(names, results[1], results[0])):
        assert a.dtype == b.dtype and _off(a, b) <= bound * (1 if i < 2 else 4), (name, _off(a, b))


def test_tokens_one_by_one_are_the_block():
    """The decode form: one token a call carries state and history on through the step kernel."""
    from vesper.column import set_scan

    layer, x, state, history = _layer()
    set_scan(layer, "fused-fp32")
    with torch.no_grad():
        whole, after, last = layer(x, state, history)
        outs = []
        for t in range(x.shape[1]):
            y, state, history = layer(x[:, t:t + 1], state, history)
            outs.append(y)
    assert _off(torch.cat(outs, 1), whole) <= 1e-5 and _off(state, after) <= 1e-5 and torch.equal(history, last)


def test_a_residual_stream_through_two_sublayers_trains():
    """norm with the residual's addition, sublayer, norm, sublayer: every parameter has a finite gradient, the same one under
    a graph's replay as in the eager step."""
    from vesper.column import set_scan
    from vesper.kernels.layer_norm import layer_norm

    first, x, state, history = _layer(seed=1)
    second = _layer(seed=2)[0]
    for layer in (first, second):
        set_scan(layer, "fused")
    gain = torch.ones(128, device=GPU, requires_grad=True)
    params = [gain, *first.parameters(), *second.parameters()]

    def work():
        y, after, _ = first(x, state, history)
        z, total = layer_norm(x, gain, residual=y)
        out, last, _ = second(z, state, history)
        loss = (total + out).square().mean() + last.square().mean() + after.square().mean()
        return [loss.detach(), *torch.autograd.grad(loss, params)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = work()
    for seed in (5, 6, 7):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in static]
        want = work()
        for a, b in zip(got, want):
            assert torch.isfinite(a).all()
            # library sums (the mean, the products) may take another order under capture: float32's own roundings
            assert _off(a, b) <= 1e-4
