"""The 8-bit norm and projections on the GPU against float64.

Bounds. The norm's scale: peak, sum of squares and root in float32, some (d / 64 / 8 + 12) roundings in
sequence: under 64 * 2^-24 of it. Codes: the kernel's y / scale carries a relative error of twice that, at most
127 * 2^-17 = 1e-3, so a code may differ from the float64 one (by one) only where the latter lies that near a
half. The product: integer sums are exact, then the sum's conversion, the scales' product and theirs are three
roundings to float32 (2^-24 each), the logistic function a few more of a value in (0, 1), and one rounding to
the output's dtype.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]

GPU = torch.device("cuda")
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_EPS = {BF16: 2.0**-8, F16: 2.0**-11, F32: 2.0**-24}
# below the smallest normal number the spacing is constant (fp16: 2^-14 * 2^-10 = 2^-24), so a rounding there is
# off by at most half of it, whatever the value
HALF_SUBNORMAL = {BF16: 2.0**-134, F16: 2.0**-25, F32: 2.0**-150}


def _norm_ref(x, residual, gain):
    s = x.double() if residual is None else x.double() + residual.double()
    y = s / torch.sqrt(s.square().mean(-1, keepdim=True) + 1e-6)
    return s, y if gain is None else y * gain.double()


def _check_norm(codes, scale, y):
    want = y.abs().amax(-1) / 127
    assert codes.dtype == torch.int8 and scale.dtype == F32
    assert bool(((scale.cpu().double() - want).abs() <= 64 * 2.0**-24 * want).all())
    t = y / want.clamp_min(1e-300)[..., None]
    got = codes.cpu().double()
    assert float((got - t).abs().max()) <= 0.5 + 1e-3
    assert int(got.abs().max()) <= 127


@pytest.mark.parametrize(("dtype", "rdtype"), [(F32, BF16), (F32, F16), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize(("m", "d"), [(1, 8), (3, 16), (5, 504), (4, 512), (7, 520), (9, 1000), (2, 1032), (6, 2048),
                                      (3, 2056), (5, 4096), (2, 4104), (3, 8192), (2, 8200), (3, 16384)])
def test_the_norm_in_8_bits(m, d, dtype, rdtype):
    from vesper.kernels.norm import rms_norm_int8

    g = torch.Generator().manual_seed(m * d)
    x = (torch.randn(m, d, generator=g) * torch.exp(2 * torch.randn(m, 1, generator=g))).to(dtype)
    residual = torch.randn(m, d, generator=g).to(rdtype)
    gain = torch.exp(0.3 * torch.randn(d, generator=g))
    for r in (None, residual):
        for gn in (None, gain):
            s, y = _norm_ref(x, r, gn)
            total = torch.empty(m, d, dtype=dtype, device=GPU) if r is not None else None
            codes, scale = rms_norm_int8(x.to(GPU), None if gn is None else gn.to(GPU),
                                         residual=None if r is None else r.to(GPU), sum_out=total)
            assert codes.shape == (m, d) and scale.shape == (m,)
            _check_norm(codes, scale, y)
            if total is not None:
                assert torch.equal(total.cpu(), (x.float() + r.float()).to(dtype))


def test_the_norm_of_edge_rows():
    """Zeros, tiny and huge rows, infinities and NaN, each alone among ordinary rows."""
    from vesper.kernels.norm import rms_norm_int8

    g = torch.Generator().manual_seed(2)
    for d in (64, 5000):
        x = torch.randn(9, d, generator=g)
        x[0] = 0
        x[1] *= 1e-30
        x[2] = x[2].clamp(-3, 3) * 1e38
        x[3, 5], x[4, 7], x[5, 9] = math.nan, math.inf, -math.inf
        x[6] = 2.5
        x[7] *= 1e-41  # subnormal
        codes, scale = rms_norm_int8(x.to(GPU))
        _, y = _norm_ref(x, None, None)
        ok = [1, 2, 6, 8]
        _check_norm(codes[ok], scale[ok], y[ok])
        assert bool(scale[3:6].isnan().all()) and not bool(codes[3:6].any())
        assert not bool(codes[[0, 7]].any()) and not bool(scale[[0, 7]].any())
    gain = torch.ones(64)
    gain[3] = math.inf
    codes, scale = rms_norm_int8(torch.randn(2, 64, generator=g).to(GPU), gain.to(GPU))
    assert bool(scale.isnan().all()) and not bool(codes.any())


def test_the_norm_takes_strided_unaligned_and_empty_input():
    from vesper.kernels.norm import rms_norm_int8

    wide = torch.randn(4, 3, 129, device=GPU)
    x = wide[..., 1:]
    a, sa = rms_norm_int8(x)
    b, sb = rms_norm_int8(x.contiguous())
    assert torch.equal(a, b) and torch.equal(sa, sb) and sa.shape == (4, 3)
    codes, scale = rms_norm_int8(torch.empty(0, 64, device=GPU))
    assert codes.shape == (0, 64) and scale.shape == (0,)


def _project_case(m, d, used, seed, cols=None):
    g = torch.Generator().manual_seed(seed)
    p, cols = len(used), cols or max(used)
    z = torch.randint(-127, 128, (m, d), generator=g, dtype=torch.int8)
    w = torch.randint(-127, 128, (p, cols, d), generator=g, dtype=torch.int8)
    zs = torch.exp(torch.randn(m, generator=g)) / 127
    ws = torch.exp(torch.randn(p, cols, generator=g)) / (127 * math.sqrt(d))
    return z, zs, w, ws


def _check_project(z, zs, w, ws, used, sig, dtype):
    from vesper.kernels.norm import projection_int8

    outs = projection_int8(z.to(GPU), zs.to(GPU), w.to(GPU), ws.to(GPU), used, sigmoid_block=sig, dtype=dtype)
    for j, (u, y) in enumerate(zip(used, outs)):
        assert y.shape == (z.shape[0], u) and y.dtype == dtype
        ref = (z.double() @ w[j, :u].double().t()) * zs.double()[:, None] * ws[j, :u].double()
        # |error| of the logistic's argument moves it by at most a quarter of that
        near = 3 * 2.0**-24 * ref.abs()
        if j == sig:
            near = near / 4 + 8 * 2.0**-24
            ref = torch.sigmoid(ref)
        assert bool(((y.cpu().double() - ref).abs() <= near + HALF_EPS[dtype] * (ref.abs() + near) + HALF_SUBNORMAL[dtype]).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize(("m", "d", "used"), [
    (1, 16, (1,)),
    (2, 48, (3, 17)),
    (16, 128, (16, 16, 16, 2)),
    (17, 144, (33, 1, 20)),
    (33, 768, (100, 100, 100, 12)),
    (64, 512, (512, 512, 512, 8)),
    (5, 4096, (300, 64, 64)),
    (65, 16, (5,)),
    (70, 240, (257, 9, 31, 3)),
    (130, 512, (512, 512, 512, 8)),
    (257, 1040, (260, 4)),
    (600, 256, (256, 256, 256, 4)),
    (1000, 768, (768, 130, 768)),
])
def test_the_projection_in_8_bits(m, d, used, dtype):
    z, zs, w, ws = _project_case(m, d, used, seed=m + d)
    _check_project(z, zs, w, ws, used, len(used) - 1 if len(used) > 1 else None, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize(("m", "used", "sig"), [(2500, (600, 250, 9), 1), (2049, (1200, 1024), None)])
def test_tiles_of_128_columns(m, used, sig, dtype):
    """Between the narrow tile (up to 256 of 128 x 64) and the wide one (over 512 of 128 x 128)."""
    z, zs, w, ws = _project_case(m, 144, used, seed=m)
    _check_project(z, zs, w, ws, used, sig, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize(("d", "sig"), [(16, 3), (272, None), (512, 0)])
def test_more_tiles_than_one_round_of_workgroups(d, sig, dtype):
    """67 x 6 tiles of 256 x 256: one, three and four stages, a last row tile of 104 tokens, ragged and narrow blocks."""
    z, zs, w, ws = _project_case(17000, d, (300, 256, 265, 9), seed=d)
    _check_project(z, zs, w, ws, (300, 256, 265, 9), sig, dtype)


@pytest.mark.parametrize("m", [3, 40, 64, 65, 300])
def test_the_largest_sums_are_exact(m):
    """Every product 127 * 127 (and its negative) over the widest row: 2.6e8, within int32."""
    d = 16384
    z = torch.full((m, d), 127, dtype=torch.int8)
    w = torch.full((1, 40, d), 127, dtype=torch.int8)
    w[0, 1::2] = -127
    _check_project(z, torch.ones(m), w, torch.ones(1, 40), (40,), None, F32)


@pytest.mark.parametrize("m", [4, 50, 200])
def test_scales_of_zero_nan_and_large_spread(m):
    from vesper.kernels.norm import projection_int8

    z, zs, w, ws = _project_case(m, 64, (20, 20), seed=4)
    zs[0], zs[1] = 0.0, math.nan
    ws[0, 3], ws[1, 5] = 0.0, 1e-30
    a, b = projection_int8(z.to(GPU), zs.to(GPU), w.to(GPU), ws.to(GPU), (20, 20), dtype=F32)
    assert not bool(a[0].any()) and bool(a[1].isnan().all()) and bool(b[1].isnan().all())
    assert not bool(a[2:, 3].any()) and bool(torch.isfinite(a[2:]).all()) and bool(torch.isfinite(b[2:]).all())


def test_weights_wider_than_used_strided_and_no_tokens():
    from vesper.kernels.norm import projection_int8

    for m in (6, 100):
        z, zs, w, ws = _project_case(m, 64, (10, 33), seed=5, cols=50)
        _check_project(z, zs, w, ws, (10, 33), None, BF16)
        want = projection_int8(z.to(GPU), zs.to(GPU), w.to(GPU), ws.to(GPU), (10, 33))
        strided = [t.to(GPU).repeat_interleave(2, -1)[..., ::2] for t in (z, zs, w, ws)]
        got = projection_int8(*strided, (10, 33))
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    z, zs, w, ws = (t.to(GPU) for t in _project_case(0, 64, (10,), seed=6))
    assert projection_int8(z, zs, w, ws, (10,))[0].shape == (0, 10)


def test_quantized_weights_are_within_half_a_step():
    from vesper.kernels.norm import quantize_weights

    w = torch.randn(3, 40, 64)
    w[1, 4] = 0
    codes, scale = quantize_weights(w.bfloat16())
    assert codes.dtype == torch.int8 and codes.shape == w.shape and scale.shape == (3, 40)
    step = scale.double()[..., None]
    assert bool(((codes.double() * step - w.bfloat16().double()).abs() <= step * (0.5 + 1e-5)).all())
    assert not bool(codes[1, 4].any()) and float(scale[1, 4]) == 0


def test_norm_then_projection_follow_the_unquantised_sublayer():
    """The pair as a sublayer uses it, against float64 of the unquantised product. The two roundings are
    uniform within half a step of each factor: an output's error has a variance of at most d (sy^2 w^2 + sw^2 y^2)
    / 12 with the steps sy, sw; six deviations bound every one of the outputs here (1.2e-9 each)."""
    from vesper.kernels.norm import projection_int8, quantize_weights, rms_norm_int8

    g = torch.Generator().manual_seed(21)
    for m in (9, 200):
        d, used = 512, (512, 512, 8)
        x, r = torch.randn(m, d, generator=g), torch.randn(m, d, generator=g).bfloat16()
        w = torch.randn(3, 512, d, generator=g) / math.sqrt(d)
        codes, scale = rms_norm_int8(x.to(GPU), residual=r.to(GPU))
        outs = projection_int8(codes, scale, *quantize_weights(w.to(GPU)), used, dtype=F32)
        _, y = _norm_ref(x, r, None)
        for j, u in enumerate(used):
            wj = w[j, :u].double()
            sy, sw = y.abs().amax(-1, keepdim=True) / 127, wj.abs().amax(-1) / 127
            var = (sy**2 * wj.square().sum(-1) + sw**2 * y.square().sum(-1, keepdim=True)) / 12 + d * (sy * sw / 12) ** 2
            assert bool(((outs[j].cpu().double() - y @ wj.t()).abs() <= 6 * var.sqrt()).all())


def test_captured_and_on_another_stream():
    from vesper.kernels.norm import projection_int8, rms_norm_int8

    for m in (8, 300):
        z, zs, w, ws = (t.to(GPU) for t in _project_case(m, 256, (256, 256), seed=8))
        x = torch.randn(m, 256, device=GPU)

        def step():
            codes, scale = rms_norm_int8(x)
            return projection_int8(codes, scale, w, ws, (256, 256))

        want = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for _ in range(3):
            graph.replay()
            fresh = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, fresh))
            x.normal_()


def test_a_product_past_32_bit_offsets():
    """More than 2^31 bytes of activations: the last rows as computed alone."""
    from vesper.kernels.norm import projection_int8

    m, d = 140_000, 16384
    z, zs, w, ws = (t.to(GPU) for t in _project_case(200, d, (24,), seed=9))
    big = torch.zeros(m, d, dtype=torch.int8, device=GPU)
    big[-200:] = z
    scales = torch.ones(m, device=GPU)
    scales[-200:] = zs
    got = projection_int8(big, scales, w, ws, (24,), dtype=F32)[0]
    assert torch.equal(got[-200:], projection_int8(z, zs, w, ws, (24,), dtype=F32)[0])
    assert not bool(got[:-200].any())


def test_refusals_on_the_gpu():
    from vesper.contracts import ContractError
    from vesper.kernels.norm import projection_int8, rms_norm_int8

    x = torch.zeros(3, 64, device=GPU)
    r = x.bfloat16()
    out = torch.empty_like(x)
    for args, match in ((dict(x=x[:, :12]), "axis 12"), (dict(x=x.double()), "dtype"), (dict(x=x, residual=x), "dtype"),
                        (dict(x=r, residual=r.half()), "dtype"), (dict(x=x, residual=r[:2]), "residual"),
                        (dict(x=x, residual=r.cpu()), "residual"), (dict(x=x, gain=torch.ones(32, device=GPU)), "gain"),
                        (dict(x=x, gain=torch.ones(64)), "gain"), (dict(x=x, sum_out=out), "residual"),
                        (dict(x=x, residual=r, sum_out=out.bfloat16()), "sum_out"), (dict(x=x, residual=r, sum_out=x), "must not be"),
                        (dict(x=r, residual=r.clone(), sum_out=r), "must not be"),
                        (dict(x=x.clone().requires_grad_()), "forward only")):
        with pytest.raises(ContractError, match=match):
            rms_norm_int8(**args)
    with torch.no_grad():
        rms_norm_int8(x, torch.ones(64, device=GPU, requires_grad=True))
    z, zs, w, ws = (t.to(GPU) for t in _project_case(3, 64, (10, 10), seed=1))
    good = dict(z=z, z_scale=zs, weights_q=w, weights_scale=ws, used=(10, 10))
    for change, match in ((dict(z=z.short()), "int8"), (dict(z=z[:, :40]), "int8"), (dict(z_scale=zs[:2]), "z_scale"),
                          (dict(z_scale=zs.half()), "z_scale"), (dict(weights_scale=ws[:1]), "weights_scale"),
                          (dict(weights_scale=ws.cpu()), "on cpu"), (dict(used=(10, 11)), "widths"), (dict(used=(10, 0)), "widths"),
                          (dict(used=(10,)), "widths"), (dict(sigmoid_block=2), "sigmoid_block"), (dict(dtype=torch.float64), "dtype")):
        with pytest.raises(ContractError, match=match):
            projection_int8(**{**good, **change})
    with pytest.raises(ContractError, match="multiple of 16"):
        projection_int8(z[:, :24], zs, w[..., :24], ws, (10, 10))


@pytest.mark.parametrize(("rows", "d"), [(2**26 + 5, 8), (2**22 + 3, 2056)])
def test_more_rows_than_one_launch_takes(rows, d):
    """Rows that repeat after 1000: each like the first of its kind, and those like a small call's."""
    from vesper.kernels.norm import rms_norm_int8

    few = torch.randn(1000, d, generator=torch.Generator().manual_seed(d)).to(torch.bfloat16).to(GPU)
    x = few.repeat((rows + 999) // 1000, 1)[:rows]
    codes, scale = rms_norm_int8(x)
    want, want_scale = rms_norm_int8(few)
    at = torch.arange(rows, device=GPU) % 1000
    assert torch.equal(scale, want_scale[at])
    for i in range(0, rows, 1000 * 2**10):
        part = codes[i:i + 1000 * 2**10]
        assert torch.equal(part, want[at[i:i + 1000 * 2**10]])


def test_more_rows_than_32_bits_count_are_refused():
    """Broadcast rows, so that nothing of that size is allocated."""
    from vesper.contracts import ContractError
    from vesper.kernels.norm import projection_int8, rms_norm_int8

    rows = 2**31
    with pytest.raises(ContractError, match="2147483647"):
        rms_norm_int8(torch.ones(1, 8, dtype=torch.bfloat16, device=GPU).expand(rows, 8))
    w = torch.ones(1, 8, 16, dtype=torch.int8, device=GPU)
    with pytest.raises(ContractError, match="2147483647"):
        projection_int8(torch.ones(1, 16, dtype=torch.int8, device=GPU).expand(rows, 16),
                        torch.ones(1, device=GPU).expand(rows), w, torch.ones(1, 8, device=GPU), (8,))


def test_a_sum_that_overlaps_an_input_in_part_is_refused():
    from vesper.contracts import ContractError
    from vesper.kernels.norm import rms_norm_int8

    n, d = 40, 64
    buf, r = torch.randn((n + 1) * d, device=GPU), torch.randn(n, d, device=GPU).bfloat16()
    x, late = buf[:n * d].view(n, d), buf[d:].view(n, d)
    before = buf.clone()
    for kwargs in (dict(x=x, residual=r, sum_out=late), dict(x=late, residual=r, sum_out=x),
                   dict(x=x.clone(), residual=buf.view(BF16)[d:(n + 1) * d].view(n, d), sum_out=x),
                   dict(x=x.clone(), residual=r, gain=buf[n * d:], sum_out=late)):
        with pytest.raises(ContractError, match="overlap"):
            rms_norm_int8(**kwargs)
    assert torch.equal(buf, before)
    # neighbours are taken, and so is a sum over an input that is read as a copy
    pair = torch.randn(2, n, d, device=GPU)
    want = pair[0] + r.float()
    rms_norm_int8(pair[0], residual=r, sum_out=pair[1])
    assert torch.equal(pair[1], want)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize(("m", "d", "used", "sig"), [
    (17, 16, (4200,), None),
    (17, 1040, (2500, 1700, 9), 2),
    (31, 144, (4097, 33), 1),
    (32, 512, (2064, 2064), 0),
    (33, 144, (2500, 1700, 9), 2),
    (48, 128, (4160, 1, 31, 16), 3),
    (63, 2064, (4111,), 0),
    (64, 512, (1500, 1500, 1500, 12), 3),
])
def test_few_tokens_against_many_columns(m, d, used, sig, dtype):
    """17 to 64 tokens against more than 256 tiles of 16 columns: workgroups of 32 columns, the last ones ragged."""
    assert sum((u + 15) // 16 for u in used) > 256
    z, zs, w, ws = _project_case(m, d, used, seed=m + d)
    _check_project(z, zs, w, ws, used, sig, dtype)


@pytest.mark.parametrize("m", [20, 50])
def test_few_tokens_against_many_wider_weights(m):
    """Columns past the used ones do not reach the outputs."""
    from vesper.kernels.norm import projection_int8

    used = (2100, 2050)
    z, zs, w, ws = _project_case(m, 144, used, seed=m, cols=2300)
    _check_project(z, zs, w, ws, used, None, F16)
    for j, u in enumerate(used):
        w[j, u:], ws[j, u:] = 77, math.nan
    want = projection_int8(z.to(GPU), zs.to(GPU), w[:, :2100].contiguous().to(GPU), ws[:, :2100].contiguous().to(GPU), used)
    for a, b in zip(projection_int8(z.to(GPU), zs.to(GPU), w.to(GPU), ws.to(GPU), used), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_the_most_tokens(dtype):
    """2^31 - 1 tokens: the last tile ends one row short of 2^31, and the rows of its last wave are the call's last."""
    from vesper.kernels.norm import projection_int8

    m, d, tail = 2**31 - 1, 16, 700
    if torch.cuda.mem_get_info()[0] < 120 * 2**30:
        pytest.skip("needs 120 GiB of free GPU memory")
    z, zs, w, ws = (t.to(GPU) for t in _project_case(tail, d, (8,), seed=31))
    big, scales = torch.empty(m, d, dtype=torch.int8, device=GPU), torch.empty(m, device=GPU)
    big[-tail:], scales[-tail:] = z, zs
    got = projection_int8(big, scales, w, ws, (8,), dtype=dtype)[0]
    assert torch.equal(got[-tail:], projection_int8(z, zs, w, ws, (8,), dtype=dtype)[0])
    del big, scales, got
    torch.cuda.empty_cache()
