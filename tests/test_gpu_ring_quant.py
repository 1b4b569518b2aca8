"""The KV ring in four bits on the GPU: tokens written, read back and attended, against float64 (``oracle.quant``).

Bounds. Codes: the kernel's quotient carries two float32 roundings (the difference and the division, each half
a step, 2^-24, of at most 15), so a code may differ from the float64 one only where the latter lies within
15 * 2^-23 < 2e-6 of a half. Scales and minima are exact in the ring's dtype. Values read back: one rounding.

Attention: one rounding to the output's dtype (half a step: eps / 2 of the value), and float32 arithmetic: the
scores' sums run over products of up to 143 |q_e| (128 + code) in units of the scale, each of some eight
roundings at the size of the whole sum, 8 * 2^-24 * 143 s sum|q| / sqrt(dk) = es; weights move by a relative
2 es (numerator and sum), and the weights times the values' scales are held in 16 bits (2^-16) with the
values' 128 taken out again, (143 s') 2^-16 at most, s' the largest scale of the values.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import needs_gpu
from oracle.quant import quant_ring_attend, quantize_rows, ring_values, row_values, unpack_rows

pytestmark = [pytest.mark.gpu, needs_gpu]

GPU = torch.device("cuda")
BF16, F16 = torch.bfloat16, torch.float16
HALF_EPS = {BF16: 2.0**-8, F16: 2.0**-11}


def _rows(g, *shape, dtype):
    x = torch.randn(*shape, generator=g) + 0.5 * torch.randn(shape[-1], generator=g)
    return x.to(dtype)


def _ring(b, hkv, dk, w, dtype):
    from vesper.kernels.ring_quant import quant_ring_empty

    return quant_ring_empty(b, hkv, dk, w, dtype, GPU)


def _clone(ring):
    from vesper.kernels.ring_quant import QuantRingKVCache

    return QuantRingKVCache(*(t.clone() for t in ring.tensors()), ring.window)


def _write(k, v, pos, ring, **kw):
    from vesper.kernels.ring_quant import quant_ring_write

    lengths = kw.pop("lengths", None)
    return quant_ring_write(k.to(GPU), v.to(GPU), pos.to(GPU), ring,
                            lengths=None if lengths is None else lengths.to(GPU), **kw)


def _check_rows(x, packed, pair):
    """Rows ``x`` (cpu) against their stored codes and pairs (cpu)."""
    codes, scale, lo, t = quantize_rows(x)
    got = unpack_rows(packed)
    assert torch.equal(pair[..., 0:1].double(), scale) and torch.equal(pair[..., 1:2].double(), lo)
    near = ((t - torch.floor(t) - 0.5).abs() < 2e-6) & (scale > 0)
    assert torch.equal(torch.where(near, codes, got), codes)
    assert float((got - t)[scale.expand_as(t) > 0].abs().max() if bool((scale > 0).any()) else 0) <= 0.5 + 15 * 2.0**-8


SIZES = [
    # b, n, w, hkv, dk
    (1, 1, 1, 1, 8),
    (2, 5, 7, 3, 16),
    (1, 33, 32, 2, 24),
    (3, 31, 100, 1, 40),
    (2, 130, 64, 8, 64),
    (2, 65, 65, 2, 72),
    (1, 77, 50, 4, 96),
    (2, 9, 200, 2, 128),
    (1, 40, 33, 1, 200),
    (2, 17, 40, 3, 256),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("b", "n", "w", "hkv", "dk"), SIZES)
def test_a_chunk_is_quantised_into_its_slots_and_read_back(b, n, w, hkv, dk, dtype):
    from vesper.kernels.ring_quant import quant_ring_read

    g = torch.Generator().manual_seed(n * dk + b)
    k, v = _rows(g, b, n, hkv, dk, dtype=dtype), _rows(g, b, n, hkv, dk, dtype=dtype)
    start = torch.randint(0, 3 * w, (b, 1), generator=g)
    pos = start + torch.arange(n)
    ring = _write(k, v, pos, _ring(b, hkv, dk, w, dtype))
    kept = min(n, w)
    last = pos[:, n - kept:]
    for i in range(b):
        at = last[i] % w
        for x, packed, pair in ((k, ring.k, ring.k_scale), (v, ring.v, ring.v_scale)):
            _check_rows(x[i, n - kept:].transpose(0, 1), packed[i].cpu()[:, at], pair[i].cpu()[:, at])
        assert torch.equal(ring.pos[i].cpu()[at], last[i]) and bool(ring.valid[i].cpu()[at].all())
        assert int(ring.valid[i].sum()) == kept
    # read back in another order, with a repeated, an absent and a negative position
    asked = torch.cat([last.flip(1), last[:, :1], last[:, -1:] + 1, last[:, :1] - 1 - w, torch.full((b, 1), -3)], 1)
    rk, rv, found = quant_ring_read(ring, asked.to(GPU))
    want = torch.ones_like(asked, dtype=torch.bool)
    want[:, kept + 1:] = False
    assert torch.equal(found.cpu(), want)
    for i in range(b):
        at = asked[i] % w
        for got, packed, pair in ((rk, ring.k, ring.k_scale), (rv, ring.v, ring.v_scale)):
            ref = ring_values(packed[i].cpu()[:, at], pair[i].cpu()[:, at]).transpose(0, 1).to(dtype)
            ref[~want[i]] = 0
            assert torch.equal(got[i].cpu(), ref)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_equal_features_of_every_size_have_a_scale_and_codes_of_zero(dtype):
    top = torch.finfo(dtype).max
    sizes = [0.0, 1e-7, 1.0, -3.0, 6e4] + ([1e-40, 1e13, -5e15, 1e30, top, -top] if dtype == BF16 else [top, -top])
    x = torch.tensor(sizes, dtype=torch.float64).to(dtype)[None, :, None, None].expand(1, len(sizes), 2, 24)
    ring = _write(x, x, torch.arange(len(sizes))[None], _ring(1, 2, 24, len(sizes), dtype))
    for packed, pair in ((ring.k, ring.k_scale), (ring.v, ring.v_scale)):
        assert not bool(packed.any()) and not bool(pair[..., 0].any())
        assert torch.equal(pair[..., 1].cpu(), x[..., 0].transpose(1, 2))
    q = x[:, :1].contiguous()
    _, ring = _attend(q, q, q, torch.zeros(1, 1, dtype=torch.long), ring)
    for size in sizes:
        k = torch.full((1, 1, 2, 24), size, dtype=torch.float64).to(dtype)
        _, out = _attend(q, k, k, torch.full((1, 1), 2 * len(sizes)), ring)
        assert not bool(out.k[:, :, 0].any()) and not bool(out.v[:, :, 0].any())


@pytest.mark.parametrize("inplace", [False, True])
def test_a_padded_batch_writes_each_rows_own_tokens_and_nothing_else(inplace):
    b, n, w, hkv, dk = 5, 20, 12, 2, 32
    g = torch.Generator().manual_seed(3)
    k, v = _rows(g, b, n, hkv, dk, dtype=BF16), _rows(g, b, n, hkv, dk, dtype=BF16)
    lengths = torch.tensor([0, 1, 12, 20, 7])
    pos = torch.tensor([[4], [0], [9], [100], [2**40]]) + torch.arange(n)
    pos[1, 1:] = -7  # what lies behind a row's end is not looked at
    ring = _ring(b, hkv, dk, w, BF16)
    for t in (ring.k, ring.v):
        t.fill_(0xA5)
    for t in (ring.k_scale, ring.v_scale):
        t.fill_(3.25)
    ring.pos.fill_(-9)
    before = _clone(ring)
    for lens in (lengths, lengths.int()):
        out = _write(k, v, pos, _clone(ring) if inplace else ring, lengths=lens, inplace=inplace)
        for i in range(b):
            m = int(lengths[i])
            kept = min(m, w)
            at = pos[i, m - kept:m] % w
            rest = torch.ones(w, dtype=torch.bool)
            rest[at] = False
            assert torch.equal(out.valid[i].cpu(), ~rest)
            assert torch.equal(out.pos[i].cpu()[at], pos[i, m - kept:m])
            for x, packed, pair in ((k, out.k, out.k_scale), (v, out.v, out.v_scale)):
                if kept:
                    _check_rows(x[i, m - kept:m].transpose(0, 1), packed[i].cpu()[:, at], pair[i].cpu()[:, at])
            for mine, old in zip(out.tensors()[:4], before.tensors()[:4]):
                assert torch.equal(mine[i].cpu()[:, rest], old[i].cpu()[:, rest])
            assert torch.equal(out.pos[i].cpu()[rest], before.pos[i].cpu()[rest])
        for mine, old in zip(ring.tensors(), before.tensors()):
            assert torch.equal(mine, old)  # the given ring is left as it was


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_at_the_edges_of_the_type(dtype):
    from vesper.kernels.ring_quant import quant_ring_read

    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    dk = 16
    base = torch.linspace(-1, 1, dk, dtype=torch.float64)
    rows = torch.stack([
        torch.zeros(dk, dtype=torch.float64), torch.full((dk,), 7.0, dtype=torch.float64), base * top, base * tiny,
        torch.where(base > 0, top, 0.0 * base), 1000 + base, torch.eye(dk, dtype=torch.float64)[3] * top]).to(dtype)
    bad = rows[1:4].clone()
    bad[0, 5], bad[1, 2], bad[2, 15] = math.nan, math.inf, -math.inf
    x = torch.cat([rows, bad]).view(1, -1, 1, dk)
    n = x.shape[1]
    ring = _write(x, x.flip(1), torch.arange(n)[None], _ring(1, 1, dk, n, dtype))
    _check_rows(rows[None], ring.k.cpu()[0, :, :7], ring.k_scale.cpu()[0, :, :7])
    assert bool(ring.k_scale[0, 0, 7:].isnan().all()) and not bool(ring.k[0, 0, 7:].any())
    k, v, found = quant_ring_read(ring, torch.arange(n, device=GPU)[None])
    assert bool(found.all()) and torch.equal(k.isnan(), v.flip(1).isnan())
    assert bool(k[0, 7:].isnan().all())
    good = k[0, :7, 0].cpu()
    assert bool(torch.isfinite(good).all())
    codes, scale, lo, _ = quantize_rows(rows)
    ref = row_values(codes, scale, lo).clamp(-top, top).to(dtype)
    assert torch.equal(good, ref)


def test_strided_and_unaligned_tokens_are_taken():
    b, n, w, hkv, dk = 2, 6, 8, 2, 64
    g = torch.Generator().manual_seed(8)
    wide = _rows(g, b, n, hkv, 2 * dk + 1, dtype=BF16).to(GPU)
    k, v = wide[..., 1:dk + 1], wide[..., dk + 1:]
    pos = torch.arange(n, device=GPU)[:, None].expand(n, b).t()
    a = _write(k, v, pos, _ring(b, hkv, dk, w, BF16))
    c = _write(k.contiguous(), v.contiguous(), pos.contiguous(), _ring(b, hkv, dk, w, BF16))
    for x, y in zip(a.tensors(), c.tensors()):
        assert torch.equal(x, y)


# ---- attention ----------------------------------------------------------------------------------


def _case(b, w, hkv, group, dk, dtype, seed, fill=1.0, base=0):
    """A ring written by ``quant_ring_write`` up to each row's own position, and the new token."""
    g = torch.Generator().manual_seed(seed)
    seen = torch.randint(int(fill * w), max(int(fill * w) + 1, 2 * w), (b, 1), generator=g)
    n = int(seen.max())
    k, v = _rows(g, b, n, hkv, dk, dtype=dtype), _rows(g, b, n, hkv, dk, dtype=dtype)
    pos = base + torch.arange(n).expand(b, n)
    ring = _ring(b, hkv, dk, w, dtype)
    if n:
        ring = _write(k, v, pos, ring, lengths=seen[:, 0])
    q = torch.randn(b, 1, hkv * group, dk, generator=g).to(dtype)
    kn, vn = _rows(g, b, 1, hkv, dk, dtype=dtype), _rows(g, b, 1, hkv, dk, dtype=dtype)
    return q, kn, vn, base + seen, ring


def _bound(q, ring, v, ref, dtype):
    dk = q.shape[-1]
    f = lambda t: float(torch.nan_to_num(t.double()).abs().max()) if t.numel() else 0.0  # noqa: E731
    sk, sv = f(ring.k_scale[..., 0]), f(ring.v_scale[..., 0])
    top = max(f(v), f(ring.v_scale[..., 1]) + 15 * sv)
    es = 8 * 2.0**-24 * 143 * sk * float(q.double().abs().sum(-1).max()) / math.sqrt(dk)
    return HALF_EPS[dtype] * ref.abs() + 2 * es * top + 143 * sv * 2.0**-16 + 2.0**-20


def _attend(q, k, v, pos, ring, **kw):
    from vesper.kernels.ring_quant import quant_ring_attention

    return quant_ring_attention(q.to(GPU), k.to(GPU), v.to(GPU), pos.to(GPU), ring, **kw)


def _reference(q, k, v, pos, ring):
    keys, values = ring_values(ring.k.cpu(), ring.k_scale.cpu()), ring_values(ring.v.cpu(), ring.v_scale.cpu())
    return quant_ring_attend(q.cpu(), k.cpu(), v.cpu(), pos.cpu(), keys, values, ring.pos.cpu(), ring.valid.cpu(), ring.window)


ATTN = [
    # b, w, hkv, group, dk, fill
    (1, 1, 1, 1, 8, 1.0),
    (3, 2, 2, 3, 16, 0.0),
    (2, 31, 1, 8, 24, 1.0),
    (2, 32, 2, 1, 32, 0.5),
    (2, 33, 2, 2, 40, 1.0),
    (1, 512, 8, 1, 64, 1.0),
    (5, 129, 4, 3, 64, 0.1),
    (2, 100, 2, 4, 72, 1.0),
    (2, 200, 2, 5, 96, 0.7),
    (1, 1000, 2, 4, 128, 1.0),
    (1, 260, 1, 7, 136, 1.0),
    (2, 300, 1, 2, 200, 1.0),
    (2, 97, 3, 6, 256, 0.9),
    (1, 4097, 1, 2, 64, 1.0),
    (300, 40, 4, 1, 64, 0.5),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("b", "w", "hkv", "group", "dk", "fill"), ATTN)
def test_attention_over_the_ring(b, w, hkv, group, dk, fill, dtype):
    q, k, v, pos, ring = _case(b, w, hkv, group, dk, dtype, seed=w + dk, fill=fill)
    ref = _reference(q, k, v, pos, ring)
    before = _clone(ring)
    o, out = _attend(q, k, v, pos, ring)
    err = (o.cpu().double() - ref).abs()
    assert bool((err <= _bound(q, ring, v, ref, dtype)).all()), float((err / _bound(q, ring, v, ref, dtype)).max())
    for mine, old in zip(ring.tensors(), before.tensors()):
        assert torch.equal(mine, old)
    # the ring that comes back: the token in its slot as a chunk of one writes it, all else as it was
    from vesper.kernels.ring_quant import quant_ring_write

    wrote = quant_ring_write(k.to(GPU), v.to(GPU), pos.to(GPU), ring)
    for mine, theirs in zip(out.tensors(), wrote.tensors()):
        assert torch.equal(mine, theirs)
    # a step repeated on the ring it wrote, in place, gives the same output
    o2, out2 = _attend(q, k, v, pos, out, inplace=True)
    assert out2 is out and torch.equal(o2, o)
    for mine, theirs in zip(out.tensors(), wrote.tensors()):
        assert torch.equal(mine, theirs)


def test_only_the_new_token_where_no_slot_is_seen():
    """Rows whose ring holds nothing, only flags that are off, only positions out of the window or ahead of the
    token, or a negative position: the output is the new token's value, whatever the unseen rows hold."""
    b, w, hkv, dk = 4, 70, 2, 64
    q, k, v, _, ring = _case(b, w, hkv, 2, dk, BF16, seed=5)
    pos = torch.tensor([[500], [500], [500], [500]])
    ring.pos[0], ring.valid[0] = 490, False
    ring.pos[1], ring.valid[1] = 430, True  # p - w
    ring.pos[2], ring.valid[2] = 501, True
    ring.pos[3], ring.valid[3] = -(2**62), True
    ring.k_scale.fill_(math.nan)
    ring.v_scale.fill_(math.inf)
    ring.k.fill_(255)
    o, _ = _attend(q, k, v, pos, ring)
    assert torch.equal(o.cpu(), v.repeat_interleave(2, dim=2))


def test_unseen_rows_of_any_contents_do_not_reach_the_output():
    b, w, hkv, dk = 3, 150, 2, 64
    for dtype in (BF16, F16):
        q, k, v, pos, ring = _case(b, w, hkv, 2, dk, dtype, seed=6, fill=0.4)
        want, _ = _attend(q, k, v, pos, ring)
        unseen = ~ring.valid | (torch.arange(w, device=GPU) == pos.to(GPU) % w)
        for t, fills in ((ring.k_scale, (math.nan, math.inf)), (ring.v_scale, (math.inf, -math.inf)), (ring.k, (255,)), (ring.v, (255,))):
            for i, x in enumerate(fills):
                part = t[..., i] if len(fills) == 2 else t
                mask = unseen[:, None, :] if len(fills) == 2 else unseen[:, None, :, None]
                part.copy_(torch.where(mask, torch.full_like(part, x), part))
        got, _ = _attend(q, k, v, pos, ring)
        assert torch.equal(got, want)


def test_a_nan_row_that_is_seen_is_attended_as_nan():
    q, k, v, pos, ring = _case(2, 64, 2, 1, 64, BF16, seed=7, fill=1.0)
    slot = int((pos[0, 0] - 3) % 64)
    ring.k_scale[0, 1, slot] = math.nan
    o, _ = _attend(q, k, v, pos, ring)
    assert bool(o[0, 0, 1].isnan().all()) and bool(torch.isfinite(o[0, 0, 0]).all()) and bool(torch.isfinite(o[1]).all())


def test_inactive_rows_give_zeros_and_are_written():
    q, k, v, pos, ring = _case(3, 64, 2, 2, 32, BF16, seed=9)
    active = torch.tensor([True, False, True], device=GPU)
    want, ring_want = _attend(q, k, v, pos, ring)
    o, out = _attend(q, k, v, pos, ring, active=active)
    assert not bool(o[1].any()) and torch.equal(o[0], want[0]) and torch.equal(o[2], want[2])
    for mine, theirs in zip(out.tensors(), ring_want.tensors()):
        assert torch.equal(mine, theirs)


def test_positions_past_32_bits():
    q, k, v, pos, ring = _case(2, 65, 2, 2, 64, BF16, seed=10, base=2**40 + 12345)
    ref = _reference(q, k, v, pos, ring)
    o, out = _attend(q, k, v, pos, ring)
    assert bool(((o.cpu().double() - ref).abs() <= _bound(q, ring, v, ref, BF16)).all())
    assert int(out.pos.max()) == int(pos.max())


def test_large_and_small_magnitudes():
    """Queries and keys of a large spread (one score far above the rest) and values of tiny scale."""
    for dtype in (BF16, F16):
        q, k, v, pos, ring = _case(2, 200, 2, 4, 64, dtype, seed=11)
        g = torch.Generator().manual_seed(12)
        n = 200
        keys, values = 6 * torch.randn(2, n, 2, 64, generator=g), 1e-4 * torch.randn(2, n, 2, 64, generator=g)
        ring = _write(keys.to(dtype), values.to(dtype), torch.arange(n).expand(2, n), ring)
        pos = torch.full((2, 1), n)
        q, k, v = 3 * q, 6 * k, (1e-4 * v.float()).to(dtype)
        ref = _reference(q, k, v, pos, ring)
        o, _ = _attend(q, k, v, pos, ring)
        err = (o.cpu().double() - ref).abs()
        assert bool((err <= _bound(q, ring, v, ref, dtype) - 2.0**-20 + 2.0**-25).all())


def test_steps_after_a_prompt_follow_the_reference():
    """A padded batch of prompts, then tokens one by one, the ring in place throughout."""
    b, n, w, hkv, dk, dtype = 3, 40, 24, 2, 64, BF16
    g = torch.Generator().manual_seed(13)
    k, v = _rows(g, b, n + 30, hkv, dk, dtype=dtype), _rows(g, b, n + 30, hkv, dk, dtype=dtype)
    lengths = torch.tensor([40, 3, 17])
    ring = _write(k[:, :n], v[:, :n], torch.arange(n).expand(b, n), _ring(b, hkv, dk, w, dtype), lengths=lengths)
    for t in range(30):
        pos = (lengths + t)[:, None]
        q = torch.randn(b, 1, hkv * 2, dk, generator=g).to(dtype)
        kn, vn = k[:, n + t:n + t + 1], v[:, n + t:n + t + 1]
        ref = _reference(q, kn, vn, pos, ring)
        tol = _bound(q, ring, vn, ref, dtype)
        o, same = _attend(q, kn, vn, pos, ring, inplace=True)
        assert same is ring
        assert bool(((o.cpu().double() - ref).abs() <= tol).all())


def test_a_captured_step_replays_as_the_eager_one():
    """Several replays at advancing positions, with eager calls of the same shape between them."""
    for b, w, hkv in ((2, 96, 2), (1, 2000, 1)):  # one workgroup a head, and a window shared by several
        q, k, v, pos, ring = (x if not isinstance(x, torch.Tensor) else x.to(GPU) for x in _case(b, w, hkv, 2, 64, BF16, seed=14))
        mine, other = _clone(ring), _clone(ring)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            _attend(q, k, v, pos, other, inplace=True, check_positions=False)
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, _ = _attend(q, k, v, pos, mine, inplace=True, check_positions=False)
        check = _clone(ring)
        for t in range(4):
            graph.replay()
            want, _ = _attend(q, k, v, pos, check, inplace=True)
            torch.cuda.synchronize()
            assert torch.equal(o, want)
            for x, y in zip(mine.tensors(), check.tensors()):
                assert torch.equal(x, y)
            pos.add_(1)
            q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(t)).to(BF16))


def test_calls_on_another_stream_and_two_at_once():
    q, k, v, pos, ring = _case(1, 3000, 2, 2, 64, BF16, seed=15)
    args = [t.to(GPU) for t in (q, k, v, pos)]
    want, _ = _attend(*args, ring)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(_attend(*args, ring, check_positions=False)[0])
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)


def test_the_last_row_of_a_cache_past_four_gibibytes():
    b, w, hkv, dk = 17, 1 << 20, 2, 256
    assert b * hkv * w * dk // 2 > 2**32
    ring = _ring(b, hkv, dk, w, BF16)
    g = torch.Generator().manual_seed(16)
    n = 37
    k, v = _rows(g, 1, n, hkv, dk, dtype=BF16), _rows(g, 1, n, hkv, dk, dtype=BF16)
    lengths = torch.zeros(b, dtype=torch.long)
    lengths[-1] = n
    start = 3 * w - 20  # the chunk wraps round the ring's end
    _write(k.expand(b, n, hkv, dk), v.expand(b, n, hkv, dk), (start + torch.arange(n)).expand(b, n), ring, lengths=lengths,
           inplace=True)
    q = torch.randn(b, 1, 2 * hkv, dk, generator=g).to(BF16)
    kn, vn = _rows(g, b, 1, hkv, dk, dtype=BF16), _rows(g, b, 1, hkv, dk, dtype=BF16)
    o, _ = _attend(q, kn, vn, torch.full((b, 1), start + n), ring, inplace=True)
    assert torch.equal(o[:-1].cpu(), vn[:-1].repeat_interleave(2, dim=2))
    small = _write(k, v, (100 + torch.arange(n))[None], _ring(1, hkv, dk, 64, BF16))
    ref = _reference(q[-1:], kn[-1:], vn[-1:], torch.full((1, 1), 100 + n), small)
    assert bool(((o[-1:].cpu().double() - ref).abs() <= _bound(q, small, vn, ref, BF16)).all())
    assert int(ring.pos[-1].max()) == start + n and int(ring.valid.sum()) == n + b


def test_one_score_far_below_the_others_and_none_above():
    """The new token alone with a score of -1e33 (its weight is still 1), and beside a ring whose scores are 0."""
    for w in (40, 5000):
        ring = _ring(1, 1, 64, w, BF16)
        q = torch.full((1, 1, 2, 64), -1e16, dtype=BF16)
        k, v = torch.full((1, 1, 1, 64), 1e16, dtype=BF16), torch.randn(1, 1, 1, 64).to(BF16)
        pos = torch.full((1, 1), 3 * w)
        o, _ = _attend(q, k, v, pos, ring)
        assert torch.equal(o.cpu(), v.repeat_interleave(2, dim=2))
        zeros, values = torch.zeros(1, w, 1, 64, dtype=BF16), torch.randn(1, w, 1, 64).to(BF16)
        ring = _write(zeros, values, pos - w + torch.arange(w), ring)
        ref = _reference(q, k, v, pos, ring)
        o, _ = _attend(q, k, v, pos, ring)
        assert bool(((o.cpu().double() - ref).abs() <= _bound(torch.zeros(1, 1, 1, 64), ring, v, ref, BF16)).all())


def test_scores_that_are_all_far_below_zero_keep_their_order():
    """Scores of -2e32 in every slot but one, -4e31 there and -2e33 of the new token: that slot's value. Equal features
    have a scale of 0, and gaps of 1e32 leave one weight, so the scores' rounding does not count."""
    for w in (40, 5000):
        pos = torch.full((1, 1), 3 * w)
        keys = torch.full((1, w, 1, 64), 5e15, dtype=BF16)
        keys[0, 2 * w // 3] = 1e15
        values = torch.randn(1, w, 1, 64, generator=torch.Generator().manual_seed(w)).to(BF16)
        ring = _write(keys, values, pos - w + torch.arange(w), _ring(1, 1, 64, w, BF16))
        q = torch.full((1, 1, 2, 64), -5e15, dtype=BF16)
        k, v = torch.full((1, 1, 1, 64), 5e16, dtype=BF16), torch.randn(1, 1, 1, 64).to(BF16)
        ref = _reference(q, k, v, pos, ring)
        o, _ = _attend(q, k, v, pos, ring)
        assert bool(((o.cpu().double() - ref).abs() <= _bound(torch.zeros(1, 1, 1, 64), ring, v, ref, BF16)).all())


def test_rings_that_are_strided_are_copied_and_refused_in_place():
    from vesper.contracts import ContractError
    from vesper.kernels.ring_quant import QuantRingKVCache, quant_ring_read

    q, k, v, pos, ring = _case(2, 48, 2, 2, 64, BF16, seed=17)
    strided = QuantRingKVCache(*(torch.stack([t, t], -1)[..., 0] for t in ring.tensors()), ring.window)
    want, ring_want = _attend(q, k, v, pos, ring)
    o, out = _attend(q, k, v, pos, strided)
    assert torch.equal(o, want)
    for mine, theirs in zip(out.tensors(), ring_want.tensors()):
        assert torch.equal(mine, theirs)
    asked = pos.to(GPU) - 1 - torch.arange(10, device=GPU)
    for a, b in zip(quant_ring_read(strided, asked), quant_ring_read(ring, asked)):
        assert torch.equal(a, b)
    for call in (lambda: _attend(q, k, v, pos, strided, inplace=True), lambda: _write(k, v, pos, strided, inplace=True)):
        with pytest.raises(ContractError, match="contiguous"):
            call()


def test_refusals_on_the_gpu():
    from vesper.contracts import ContractError
    from vesper.kernels.ring_quant import QuantRingKVCache, quant_ring_attention, quant_ring_read, quant_ring_write

    ring = _ring(2, 2, 16, 8, BF16)
    x = torch.zeros(2, 3, 2, 16, dtype=BF16, device=GPU)
    pos = torch.arange(3, device=GPU).expand(2, 3)
    for bad, match in ((pos - 1, "nonnegative"), (pos * 2, "consecutive"), (pos.flip(1), "consecutive")):
        with pytest.raises(ContractError, match=match):
            quant_ring_write(x, x, bad, ring)
    for lengths in ([-1, 2], [2, 4]):
        with pytest.raises(ContractError, match="lengths"):
            quant_ring_write(x, x, pos, ring, lengths=torch.tensor(lengths, device=GPU))
    with pytest.raises(ContractError, match="lengths"):
        quant_ring_write(x, x, pos, ring, lengths=torch.tensor([1, 2]))
    with pytest.raises(ContractError, match="axis"):
        quant_ring_write(x, x, pos, ring, lengths=torch.tensor([1, 2, 3], device=GPU))
    with pytest.raises(ContractError, match="forward only"):
        quant_ring_write(x.clone().requires_grad_(), x, pos, ring)
    one, at = x[:, :1], pos[:, :1]
    with pytest.raises(ContractError, match="forward only"):
        quant_ring_attention(one.clone().requires_grad_(), one, one, at, ring)
    with torch.no_grad():
        quant_ring_attention(one.clone().requires_grad_(), one, one, at, ring)
    with pytest.raises(ContractError, match="nonnegative"):
        quant_ring_attention(one, one, one, at - 1, ring)
    with pytest.raises(ContractError, match="at most 8"):
        quant_ring_attention(one.repeat(1, 1, 9, 1), one, one, at, ring)
    with pytest.raises(ContractError, match="need a multiple"):
        quant_ring_attention(one[:, :, :1], one, one, at, ring)
    with pytest.raises(ContractError, match="active"):
        quant_ring_attention(one, one, one, at, ring, active=torch.ones(2, dtype=torch.bool))
    with pytest.raises(ContractError, match="cache.pos is on cpu"):
        quant_ring_attention(one, one, one, at, QuantRingKVCache(*ring.tensors()[:4], ring.pos.cpu(), ring.valid, 8))
    learned = QuantRingKVCache(ring.k, ring.v, ring.k_scale.clone().requires_grad_(), *ring.tensors()[3:], 8)
    with pytest.raises(ContractError, match="forward only"):
        quant_ring_read(learned, pos)
    assert not bool(ring.valid.any())  # nothing was written


def test_calls_of_no_rows_and_no_tokens():
    from vesper.kernels.ring_quant import quant_ring_attention, quant_ring_read, quant_ring_write

    for b, n in ((0, 3), (2, 0)):
        ring = _ring(b, 2, 16, 8, BF16)
        x, pos = torch.zeros(b, n, 2, 16, dtype=BF16, device=GPU), torch.zeros(b, n, dtype=torch.long, device=GPU)
        out = quant_ring_write(x, x, pos, ring)
        assert out.k.shape == ring.k.shape and not bool(out.valid.any())
        k, v, found = quant_ring_read(ring, pos)
        assert k.shape == v.shape == (b, n, 2, 16) and found.shape == (b, n)
    x = torch.zeros(0, 1, 2, 16, dtype=BF16, device=GPU)
    o, _ = quant_ring_attention(x, x, x, torch.zeros(0, 1, dtype=torch.long, device=GPU), _ring(0, 2, 16, 8, BF16))
    assert o.shape == (0, 1, 2, 16)


def test_token_counts_past_32_bits_are_refused():
    """2^32 + 8 broadcast tokens, which cut to 32 bits would be 8, against a ring that the kernels take as it is."""
    from vesper.contracts import ContractError
    from vesper.kernels.ring_quant import quant_ring_read, quant_ring_write

    n = 2**32 + 8
    tokens, pos = torch.zeros(1, dtype=BF16, device=GPU).expand(1, n, 1, 8), torch.zeros(1, dtype=torch.long, device=GPU).expand(1, n)
    ring = _ring(1, 1, 8, 4, BF16)
    with pytest.raises(ContractError, match="at most 2147483647"):
        quant_ring_write(tokens, tokens, pos, ring)
    with pytest.raises(ContractError, match="at most 2147483647"):
        quant_ring_read(ring, pos)
    assert not bool(ring.valid.any())


def test_the_most_tokens_a_row():
    """2^31 - 1 tokens, of which the last four stay: the row's end is next to the largest int."""
    n, w, dk = 2**31 - 1, 4, 8
    if torch.cuda.mem_get_info()[0] < 80 * 2**30:
        pytest.skip("needs 80 GiB of free GPU memory")
    tokens, pos = torch.empty(1, n, 1, dk, dtype=BF16, device=GPU), torch.empty(1, n, dtype=torch.long, device=GPU)
    last = torch.randn(1, w, 1, dk, generator=torch.Generator().manual_seed(30)).to(BF16)
    tokens[:, -w:], pos[:, -w:] = last.to(GPU), torch.arange(n - w, n, device=GPU)
    ring = _write(tokens, tokens, pos, _ring(1, 1, dk, w, BF16), check_positions=False)
    want = _write(last, last, torch.arange(n - w, n)[None], _ring(1, 1, dk, w, BF16))
    for mine, theirs in zip(ring.tensors(), want.tensors()):
        assert torch.equal(mine, theirs)
    assert int(ring.valid.sum()) == w
    del tokens, pos
    torch.cuda.empty_cache()
