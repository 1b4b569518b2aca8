"""Layer norm's kernels against float64: every type, widths from one to the widest, rows from one to many.

Tolerances, relative to the 2-norm: a result held in t is off by at most half a step of each value, eps(t) / 2 (bfloat16
2^-8, float16 2^-11); a row's two sums in float32 are lane sums of at most 128 terms and 10 joins, and three more
roundings follow: 150 * 2^-24 < 1e-5 of the row's values; the sums over rows are of at most 64 rows in order and 256
partial rows, 320 * 2^-24 = 2e-5 of the magnitudes summed. Where a row's mean is far larger than its deviations, their
rounding counts in units of the mean: the tests of such rows say so.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import needs_gpu
from oracle.gated import layer_norm as oracle_norm

pytestmark = [pytest.mark.gpu, needs_gpu]

GPU = torch.device("cuda")
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [(F32, F32, F32), (F32, BF16, BF16), (F32, F16, F16), (F32, BF16, F32), (F32, F32, F16), (F32, F16, BF16), (BF16, BF16, BF16),
         (F16, F16, F16)]
SIZES = [(1, 1), (5, 2), (3, 7), (4, 8), (65, 24), (1000, 33), (64, 512), (63, 520), (130, 768), (17, 1024), (9, 1032), (300, 2048),
         (10, 2050), (33, 4096), (7, 4104), (5, 8192), (3, 8200), (2, 16384), (3, 16383), (6000, 64)]


def _held(dtype):
    return torch.finfo(dtype).eps / 2 * (1 if dtype != F32 else 0) + 2e-5


def _close(got, want, what, held=None):
    got, want = got.detach().cpu().double(), want.detach().cpu().double()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    off, norm = float((got - want).norm()), float(want.norm())
    assert off <= held * norm + 1e-30, (what, off / max(norm, 1e-30))


def _inputs(m, d, x, r, y, seed=0, lead=None):
    gen = torch.Generator().manual_seed(seed)
    lead = (m,) if lead is None else lead
    t = {"x": torch.randn(*lead, d, generator=gen) * torch.exp(torch.randn(*lead, 1, generator=gen)) + torch.randn(*lead, 1, generator=gen),
         "residual": torch.randn(*lead, d, generator=gen), "gain": torch.exp(0.3 * torch.randn(d, generator=gen)),
         "bias": torch.randn(d, generator=gen), "dy": torch.randn(*lead, d, generator=gen), "ds": torch.randn(*lead, d, generator=gen)}
    types = {"x": x, "residual": r, "gain": F32, "bias": F32, "dy": y, "ds": x}
    return {n: v.to(GPU, types[n]) for n, v in t.items()}


def _want(t, eps, residual=True, bias=True, dy=True, ds=True):
    """y, s and the gradients of x, gain, bias, residual in float64."""
    leaves = {n: t[n].detach().cpu().double().requires_grad_() for n in ("x", "gain", "bias", "residual")}
    y, s = oracle_norm(leaves["x"], leaves["gain"], leaves["bias"] if bias else None, leaves["residual"] if residual else None, eps)
    loss = (y * t["dy"].cpu().double()).sum() * dy + ((s * t["ds"].cpu().double()).sum() if residual and ds else 0)
    grads = torch.autograd.grad(loss, list(leaves.values()), allow_unused=True)
    return y, s, dict(zip(leaves, grads))


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_norm_and_gradients_match_float64(types, size):
    from vesper.kernels.layer_norm import layer_norm

    m, d = size
    t = _inputs(m, d, *types, seed=m + d)
    eps = 1e-2  # rows of one or two values have deviations near zero
    leaves = [t[n].requires_grad_() for n in ("x", "gain", "bias", "residual")]
    y, s = layer_norm(t["x"], t["gain"], t["bias"], residual=t["residual"], eps=eps, dtype=types[2])
    grads = torch.autograd.grad([y, s], leaves, [t["dy"], t["ds"]])
    want_y, want_s, want = _want(t, eps)
    assert y.dtype == types[2] and s.dtype == types[0]
    _close(y, want_y, "y", _held(types[2]))
    _close(s, want_s, "sum", _held(types[0]))
    for (n, leaf), g in zip(zip(("x", "gain", "bias", "residual"), leaves), grads):
        assert g.dtype == leaf.dtype and g.shape == leaf.shape
        if d == 1 and n == "gain":  # a row of one value has no deviation
            assert float(g.abs().max()) <= 1e-30 + 2e-5 * float(t["dy"].abs().sum())
            continue
        _close(g, want[n], n, _held(leaf.dtype))
    with torch.no_grad():
        again, total = layer_norm(t["x"], t["gain"], t["bias"], residual=t["residual"], eps=eps, dtype=types[2])
    assert torch.equal(again, y) and torch.equal(total, s)


@pytest.mark.parametrize("types", [(F32, F32, F32), (F32, F32, BF16), (BF16, BF16, BF16)], ids=str)
@pytest.mark.parametrize("size", [(5, 7), (70, 768), (20, 4096)], ids=str)
@pytest.mark.parametrize("bias", [False, True])
def test_without_a_residual_and_without_a_bias(types, size, bias):
    from vesper.kernels.layer_norm import layer_norm

    t = _inputs(*size, *types, lead=(size[0], 1))
    leaves = [t[n].requires_grad_() for n in (("x", "gain", "bias") if bias else ("x", "gain"))]
    y = layer_norm(t["x"], t["gain"], t["bias"] if bias else None, dtype=types[2])
    assert y.shape == t["x"].shape
    grads = torch.autograd.grad(y, leaves, t["dy"])
    want_y, _, want = _want(t, 1e-5, residual=False, bias=bias)
    _close(y, want_y, "y", _held(types[2]))
    for n, leaf, g in zip(("x", "gain", "bias"), leaves, grads):
        _close(g, want[n], n, _held(leaf.dtype))


def test_only_one_of_the_results_is_used():
    from vesper.kernels.layer_norm import layer_norm

    t = _inputs(50, 264, F32, BF16, BF16)
    leaves = [t[n].requires_grad_() for n in ("x", "gain", "bias", "residual")]
    for which in (0, 1):
        out = layer_norm(t["x"], t["gain"], t["bias"], residual=t["residual"], dtype=BF16)[which]
        grads = torch.autograd.grad(out, leaves, t["ds"] if which else t["dy"])
        _, _, want = _want(t, 1e-5, dy=which == 0, ds=which == 1)
        for n, leaf, g in zip(("x", "gain", "bias", "residual"), leaves, grads):
            _close(g, want[n], n, _held(leaf.dtype))


def test_gradients_against_differences():
    """Central differences of the float64 norm along random ways: steps of 1e-4, off by about 1e-8."""
    from vesper.kernels.layer_norm import layer_norm

    t = _inputs(9, 40, F32, F32, F32)
    names = ("x", "gain", "bias", "residual")
    leaves = [t[n].requires_grad_() for n in names]
    grads = torch.autograd.grad(list(layer_norm(*leaves[:3], residual=leaves[3])), leaves, [t["dy"], t["ds"]])
    exact = [x.detach().cpu().double() for x in leaves]

    def loss(args):
        y, s = oracle_norm(*args, 1e-5)
        return float((y * t["dy"].cpu().double()).sum() + (s * t["ds"].cpu().double()).sum())

    gen = torch.Generator().manual_seed(3)
    for i, name in enumerate(names):
        way = torch.randn(exact[i].shape, generator=gen, dtype=torch.float64)
        ends = [loss([x + (s * 1e-4 * way if j == i else 0) for j, x in enumerate(exact)]) for s in (1, -1)]
        got = float((grads[i].cpu().double() * way).sum())
        assert abs(got - (ends[0] - ends[1]) / 2e-4) <= 3e-5 * float(grads[i].cpu().double().norm() * way.norm()), name


@pytest.mark.parametrize("types", [(F32, BF16, BF16), (F16, F16, F16)], ids=str)
def test_strided_and_unaligned_inputs_are_the_contiguous_ones(types):
    from vesper.kernels.layer_norm import layer_norm

    def other(t):
        buf = torch.zeros(t.numel() + 1, dtype=t.dtype, device=GPU)[1:].view(t.shape[::-1])
        return buf.permute(*range(t.dim())[::-1]).copy_(t)

    t = _inputs(37, 64, *types)
    results = []
    for change in (lambda v: v, other):
        leaves = [change(t[n]).detach().requires_grad_() for n in ("x", "gain", "bias", "residual")]
        y, s = layer_norm(*leaves[:3], residual=leaves[3], dtype=types[2])
        results.append([y, s, *torch.autograd.grad([y, s], leaves, [change(t["dy"]), change(t["ds"])])])
    for a, b in zip(*results):
        _close(a, b, "strided", _held(a.dtype))
    # contiguous but off 16 bytes: the kernel of single elements, whose sums run in another order
    x = torch.zeros(37 * 64 + 1, dtype=types[0], device=GPU)[1:].view(37, 64).copy_(t["x"])
    with torch.no_grad():
        _close(layer_norm(x, t["gain"], dtype=types[2]), layer_norm(t["x"], t["gain"], dtype=types[2]), "offset", 2 * _held(types[2]))


def test_rows_of_extreme_values():
    from vesper.kernels.layer_norm import layer_norm

    gen = torch.Generator().manual_seed(0)
    base = torch.randn(8, 512, generator=gen)
    x = base.clone()
    x[1] *= 2.0**100  # squares past float32
    x[2] *= 2.0**-100  # far below eps
    x[3] = 3.0  # no deviation
    x[4] = 0.0
    x[5, 7] = 2.0**125  # one huge value
    x[6, 3] = math.inf
    x[7, 3] = math.nan
    gain = torch.ones(512)
    leaf = x.to(GPU).requires_grad_()
    y = layer_norm(leaf, gain.to(GPU))
    dx, = torch.autograd.grad(y, leaf, torch.ones_like(y) + base.to(GPU))
    exact = x.double().requires_grad_()
    want, _ = oracle_norm(exact, gain.double(), None, None, 1e-5)
    want_dx, = torch.autograd.grad(want, exact, (torch.ones_like(base) + base).double())
    for i in (0, 1, 2, 5):
        _close(y[i], want[i], f"row {i}", 2e-5)
        # the gradient is w = dy less its mean and its part along the row, which is most of this dy = 1 + base (all of it in
        # row 0): of three terms of at most |w| rstd each is off by 2e-5, whatever little they leave
        rstd = 1 / math.sqrt(float(x[i].double().var(correction=0)) + 1e-5)
        off = float((dx[i].cpu().double() - want_dx[i]).norm())
        assert off <= 3 * 2e-5 * rstd * float((1 + base[i]).norm()), (i, off)
    # a mean of 512 equal values is off by a rounding or two, which 1 / sqrt(eps) = 316 magnifies
    assert float(y[3].abs().max()) <= 3 * 2.0**-23 * 3 * 317 and not bool(y[4].any())
    assert bool(torch.isnan(y[6]).any()) and bool(torch.isnan(y[7]).all())


def test_a_row_does_not_see_another():
    from vesper.kernels.layer_norm import layer_norm

    t = _inputs(40, 1000, F32, BF16, BF16)
    x = t["x"].clone()
    x[7] = math.nan
    outs = []
    for v in (x, t["x"]):
        leaf = v.detach().requires_grad_()
        y, s = layer_norm(leaf, t["gain"], t["bias"], residual=t["residual"], dtype=BF16)
        outs.append([y, s, *torch.autograd.grad([y, s], leaf, [t["dy"], t["ds"]])])
    keep = torch.arange(40, device=GPU) != 7
    for a, b in zip(*outs):
        assert torch.equal(a[keep], b[keep])


def test_captured_and_on_another_stream_and_repeated():
    from vesper.kernels.layer_norm import layer_norm

    t = _inputs(3000, 768, F32, BF16, BF16)
    names = ("x", "gain", "bias", "residual")
    leaves = [t[n].requires_grad_() for n in names]

    def work():
        y, s = layer_norm(*leaves[:3], residual=leaves[3], dtype=BF16)
        return [y.detach(), s.detach(), *torch.autograd.grad([y, s], leaves, [t["dy"], t["ds"]])]

    first = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = work()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = work()
    for seed in (1, 2, 3):
        fresh = _inputs(3000, 768, F32, BF16, BF16, seed=seed)
        with torch.no_grad():
            for n in (*names, "dy", "ds"):
                t[n].copy_(fresh[n])
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in static]
        for a, b in zip(got, work()):
            assert torch.equal(a, b)


def test_no_rows_and_a_second_derivative():
    from vesper.kernels.layer_norm import layer_norm

    x = torch.zeros(0, 64, device=GPU, requires_grad=True)
    gain = torch.ones(64, device=GPU, requires_grad=True)
    y, s = layer_norm(x, gain, residual=torch.zeros(0, 64, device=GPU, dtype=BF16), dtype=BF16)
    assert y.shape == (0, 64) and y.dtype == BF16 and s.dtype == F32
    dx, dg = torch.autograd.grad([y, s], [x, gain], [torch.zeros_like(y), torch.zeros_like(s)])
    assert dx.shape == (0, 64) and not bool(dg.any())
    x = torch.randn(4, 64, device=GPU, requires_grad=True)
    first, = torch.autograd.grad(layer_norm(x, gain).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first.sum().backward()


def test_offsets_past_32_bits():
    from vesper.kernels.layer_norm import layer_norm

    m, d = 530000, 4096  # 2.2e9 elements
    gen = torch.Generator(device=GPU).manual_seed(0)
    x = torch.empty(m, d, device=GPU, dtype=BF16).normal_(generator=gen).requires_grad_()
    gain = torch.ones(d, device=GPU)
    y = layer_norm(x, gain)
    dx, = torch.autograd.grad(y, x, x.detach())
    tail = x.detach()[-3:].clone().requires_grad_()
    small = layer_norm(tail, gain)
    assert torch.equal(y[-3:], small)
    assert torch.equal(dx[-3:], torch.autograd.grad(small, tail, tail.detach())[0])


@pytest.mark.parametrize("types", [(F32, F32, F32), (F32, BF16, F16), (BF16, BF16, BF16)], ids=str)
@pytest.mark.parametrize("size", [(3000, 513), (40, 1025), (700, 2047), (33, 4097), (9, 8191), (4, 8193), (2100, 12), (50, 5000)], ids=str)
def test_odd_and_wide_rows(types, size):
    test_norm_and_gradients_match_float64(types, size)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d", [1, 9, 513, 2051])
def test_rows_that_end_anywhere_write_no_neighbour(dtype, d):
    """The library's entries with outputs one element into larger memory: what is before and behind them stays."""
    from vesper.kernels import _lib

    m, code = 5, {F32: 0, BF16: 1, F16: 2}[dtype]
    t = _inputs(m, d, dtype, dtype, dtype, seed=d)

    def guarded(like):
        whole = torch.full((like.numel() + 40,), 7.0, dtype=like.dtype, device=GPU)
        return whole, whole[1 : 1 + like.numel()]

    outs = {n: guarded(t["x"]) for n in ("sum", "y", "dx")} | {n: guarded(t["gain"]) for n in ("dgain", "dbias")}
    stats = torch.empty(m, 2, device=GPU)
    stream = _lib.stream_of(GPU if GPU.index is not None else torch.device("cuda", torch.cuda.current_device()))
    _lib.call("vsp_layer_norm", t["x"].data_ptr(), t["residual"].data_ptr(), t["gain"].data_ptr(), t["bias"].data_ptr(),
              outs["sum"][1].data_ptr(), outs["y"][1].data_ptr(), stats.data_ptr(), code, code, code, m, d, 1e-2, stream)
    nbytes = int(_lib.library().vsp_layer_norm_backward_workspace_bytes(m, d))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=GPU)
    summed = dtype == F32  # float32 goes back from the sum
    _lib.call("vsp_layer_norm_backward", (outs["sum"][1] if summed else t["x"]).data_ptr(), None if summed else t["residual"].data_ptr(),
              t["gain"].data_ptr(), stats.data_ptr(), t["dy"].data_ptr(), t["ds"].data_ptr(), outs["dx"][1].data_ptr(), None,
              outs["dgain"][1].data_ptr(), outs["dbias"][1].data_ptr(), ws.data_ptr(), nbytes, code, code, code, m, d, stream)
    torch.cuda.synchronize()
    want_y, want_s, want = _want(t, 1e-2)
    for name, exact in (("sum", want_s), ("y", want_y), ("dx", want["x"]), ("dgain", want["gain"]), ("dbias", want["bias"])):
        whole, inner = outs[name]
        assert bool((whole[:1] == 7).all()) and bool((whole[1 + inner.numel() :] == 7).all()), name
        if d > 1 or name in ("sum", "dbias"):
            _close(inner.view(exact.shape), exact, name, _held(inner.dtype))
