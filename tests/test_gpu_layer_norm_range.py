"""Layer norm's rows over float32's range, forward and backward, against float64.

Tolerances, relative to the 2-norm: a row's sums in float32 are of at most 128 terms a lane and 10 joins, and three more
roundings follow: 150 * 2^-24 < 1e-5 of the magnitudes summed; results held in bfloat16 are off by half a step, 2^-8, more.
Rows around zero: 2e-5. Rows whose mean is ten times their deviation: the mean is off by up to 1e-5 of itself, which is 1e-4
of the deviations: 1.2e-4. The gradient of x is w = dy gain less its mean and its part along the row: three terms of at most
|w| / deviation each.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import needs_gpu
from oracle.gated import layer_norm as oracle_norm

pytestmark = [pytest.mark.gpu, needs_gpu]

GPU = torch.device("cuda")
BF16, F32 = torch.bfloat16, torch.float32


def _check(x, residual, dtype, eps, bound, grads=True):
    """The norm of ``x`` (and the residual), its sums and its gradients, each row by itself, against float64."""
    from vesper.kernels.layer_norm import layer_norm

    d = x.shape[-1]
    gen = torch.Generator().manual_seed(d)
    gain, bias, dy = torch.exp(0.3 * torch.randn(d, generator=gen)), torch.randn(d, generator=gen), torch.randn(x.shape, generator=gen)
    held = {F32: 0.0, BF16: 2.0**-8}
    leaves = [t.to(GPU).requires_grad_() for t in (x, gain, bias, *(() if residual is None else (residual,)))]
    dy = dy.to(dtype)
    out = layer_norm(*leaves[:3], residual=None if residual is None else leaves[3], eps=eps, dtype=dtype)
    y = out if residual is None else out[0]
    exact = [t.detach().cpu().double().requires_grad_() for t in leaves]
    plain, s = oracle_norm(*exact[:3], None if residual is None else exact[3], eps)
    got, want, s = y.detach().cpu().double(), plain.detach(), s.detach()
    assert torch.isfinite(got).all()
    for row in range(x.shape[0]):
        assert float((got[row] - want[row]).norm()) <= (bound + held[dtype]) * float(want[row].norm()), row
    if not grads:
        return
    dx, dgain, dbias = (t.cpu().double() for t in torch.autograd.grad(y, leaves[:3], dy.to(GPU)))
    want_dx, want_dgain, want_dbias = torch.autograd.grad(plain, exact[:3], dy.double())
    deviation = s.var(-1, correction=0, keepdim=True)
    rstd = 1 / torch.sqrt(deviation + eps)
    w = dy.double() * gain.double()
    for row in range(x.shape[0]):
        off = float((dx[row] - want_dx[row]).norm())
        assert off <= (3 * bound + held[leaves[0].dtype]) * float(rstd[row]) * float(w[row].norm()), (row, off)
    xh = (s - s.mean(-1, keepdim=True)) * rstd
    assert float((dgain - want_dgain).norm()) <= bound * float((dy.double().abs() * xh.abs()).sum(0).norm())
    assert float((dbias - want_dbias).norm()) <= 1e-5 * float(dy.double().abs().sum(0).norm())


WIDTHS = [8, 9, 317, 512, 513, 1024, 1025, 2048, 3000, 4096, 8192, 8193, 16383, 16384]


@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (BF16, BF16)], ids=str)
@pytest.mark.parametrize("d", WIDTHS)
def test_rows_whose_sum_passes_float32(types, d):
    """Below 2^126 each, 5 rows: around zero, of one sign, and a plain one between them."""
    gen = torch.Generator().manual_seed(d)
    x = torch.randn(5, d, generator=gen)
    for row, scale in ((0, 2.0**123), (3, 2.0**123)):
        x[row] *= scale
    _check(x.to(types[0]), None, types[1], 1e-5, 2e-5)
    for row, sign in ((1, 1), (4, -1)):
        x[row] = sign * 2.0**125 * (1 + 0.1 * x[row])
    _check(x.to(types[0]), None, types[1], 1e-5, 1.2e-4)


@pytest.mark.parametrize("d", [24, 513, 1024, 4096, 16384])
def test_sums_with_a_residual_that_pass_float32(d):
    gen = torch.Generator().manual_seed(d)
    x, r = 2.0**124 * (1 + 0.1 * torch.randn(3, d, generator=gen)), 2.0**124 * (1 + 0.1 * torch.randn(3, d, generator=gen))
    _check(x, r, F32, 1e-5, 1.5e-4)  # the sum's deviation is 0.14 of 2: its mean 14 times it
    _check(x.to(BF16), r.to(BF16), BF16, 1e-5, 1.5e-4)


@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (BF16, BF16)], ids=str)
@pytest.mark.parametrize("eps", [0.0, 2.0**-140])
@pytest.mark.parametrize("d", [2, 8, 513, 1024, 4096, 16384])
def test_rows_of_small_deviations_without_an_eps(types, eps, d):
    """Squares below float32 beside an eps of nothing: deviations of 2^-80 and 2^-110, and plain and large rows between."""
    x = torch.randn(5, d, generator=torch.Generator().manual_seed(d))
    x[:, ::2] += 1  # two values that differ
    for row, scale in ((0, 2.0**-80), (1, 2.0**-110), (3, 2.0**80), (4, 2.0**-40)):
        x[row] *= scale
    _check(x.to(types[0]), None, types[1], eps, 2e-5)


def test_the_smallest_rows_and_rows_without_deviations():
    from vesper.kernels.layer_norm import layer_norm

    x = torch.zeros(4, 256)
    x[0, ::2], x[1, ::2], x[2, ::2] = 2.0**-126, 2.0**-145, 1.0
    y = layer_norm(x.to(GPU), torch.ones(256, device=GPU), eps=0.0).cpu()
    want = torch.ones(256).index_fill(0, torch.arange(1, 256, 2), -1.0)  # exact: powers of two throughout
    assert torch.equal(y[:3], want.expand(3, 256)) and bool(y[3].isnan().all())
    small = layer_norm(x.to(GPU), torch.ones(256, device=GPU), eps=1e-5).cpu()
    assert float(small[1].abs().max()) < 2.0**-130 and not bool(small[3].any())


def test_a_row_of_infinities_or_nan_stays_one():
    from vesper.kernels.layer_norm import layer_norm

    x = torch.randn(4, 700, generator=torch.Generator().manual_seed(0))
    clean = layer_norm(x.to(GPU), torch.ones(700, device=GPU))
    x[1, 5], x[2, 9] = math.inf, math.nan
    y = layer_norm(x.to(GPU), torch.ones(700, device=GPU))
    assert bool(y[1].isnan().any()) and bool(y[2].isnan().all())
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3])


@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (BF16, BF16)], ids=str)
@pytest.mark.parametrize("d", [8, 264, 768, 2048, 8192])
def test_memory_at_16_but_not_32_bytes_gives_the_same_bits(types, d):
    from vesper.kernels.layer_norm import layer_norm

    def moved(t):
        buf = torch.empty(t.numel() + 32, dtype=t.dtype, device=GPU)
        first = next(i for i in range(32) if (buf.data_ptr() + i * t.element_size()) % 32 == 16)
        return buf[first : first + t.numel()].view(t.shape).copy_(t)

    gen = torch.Generator().manual_seed(d)
    t = [torch.randn(33, d, generator=gen).to(GPU, types[0]), torch.rand(d, generator=gen).to(GPU), torch.rand(d, generator=gen).to(GPU),
         torch.randn(33, d, generator=gen).to(GPU, types[0])]
    dy, ds = torch.randn(33, d, generator=gen).to(GPU, types[1]), torch.randn(33, d, generator=gen).to(GPU, types[0])
    results = []
    for change in (lambda v: v, moved):
        leaves = [change(v).detach().requires_grad_() for v in t]
        y, s = layer_norm(*leaves[:3], residual=leaves[3], dtype=types[1])
        results.append([y, s, *torch.autograd.grad([y, s], leaves, [change(dy), change(ds)])])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16)], ids=str)
@pytest.mark.parametrize("size", [(300000, 64), (40000, 513), (20001, 1024), (9000, 4096)], ids=str)
def test_sums_over_many_rows(types, size):
    """The gain's and the bias's gradients of many rows. At most 1024 workgroups, at least one a CU, 256, add up their rows in
    order (four rows at once up to 1024 wide): 300000 / 1024 = 293 rows, 4 waves, then the partial rows, sixteen waves of 64:
    8 in order in each of 8 sums, 3 joins, 16 in order. 324 roundings of 2^-24 are 2e-5 of the magnitudes summed, and each
    row's own values are off by 1e-5: 3e-5."""
    from vesper.kernels.layer_norm import layer_norm

    m, d = size
    gen = torch.Generator(GPU).manual_seed(d)
    x, dy = (torch.randn(m, d, device=GPU, generator=gen).to(t) for t in types)
    gain, bias = torch.rand(d, device=GPU, generator=gen).requires_grad_(), torch.zeros(d, device=GPU, requires_grad=True)
    dgain, dbias = torch.autograd.grad(layer_norm(x, gain, bias, dtype=types[1]), [gain, bias], dy)
    want = [torch.zeros(d, dtype=torch.float64) for _ in range(4)]
    for part in range(0, m, 10000):
        xs, gs = x[part : part + 10000].cpu().double(), dy[part : part + 10000].cpu().double()
        xh = (xs - xs.mean(-1, keepdim=True)) / torch.sqrt(xs.var(-1, correction=0, keepdim=True) + 1e-5)
        for total, term in zip(want, (gs * xh, gs, (gs * xh).abs(), gs.abs())):
            total += term.sum(0)
    assert float((dgain.cpu().double() - want[0]).norm()) <= 3e-5 * float(want[2].norm())
    assert float((dbias.cpu().double() - want[1]).norm()) <= 2e-5 * float(want[3].norm())
