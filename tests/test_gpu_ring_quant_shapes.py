"""Every form of the four-bit ring's attention over a filled ring: how many waves a workgroup has, how many workgroups
share a head's window, and the join of those, at widths of whole and of part pieces, in both types.

The rule of the forms, restated: with ``heads`` = b hkv and tiles of 32 slots, four waves a workgroup where ``heads`` is
256 or more, or where ``heads`` times the splits that the window allows (a split of at least 32 tiles up to width 64, 16
beyond) is 512 or more; else 16 waves up to width 64 and eight beyond. The join runs 256 threads up to eight splits and
1024 beyond. Bounds are those of ``test_gpu_ring_quant.py``.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import needs_gpu

GPU = torch.device("cuda")
BF16, F16 = torch.bfloat16, torch.float16
HALF_EPS = {BF16: 2.0**-8, F16: 2.0**-11}

FORMS = [
    # b, w, hkv, group, dk, waves, splits
    (32, 520, 8, 1, 8, 4, 1),
    (32, 520, 8, 3, 24, 4, 1),
    (32, 520, 8, 2, 40, 4, 1),
    (32, 520, 8, 8, 64, 4, 1),
    (32, 520, 8, 4, 72, 4, 1),
    (32, 520, 8, 5, 96, 4, 1),
    (32, 520, 8, 2, 128, 4, 1),
    (32, 520, 8, 7, 136, 4, 1),
    (32, 520, 8, 2, 200, 4, 1),
    (32, 520, 8, 6, 256, 4, 1),
    (16, 8300, 4, 2, 40, 4, 8),
    (16, 8191, 4, 3, 64, 4, 8),
    (8, 8300, 4, 2, 72, 4, 16),
    (8, 8300, 4, 4, 128, 4, 16),
    (8, 8300, 4, 1, 200, 4, 16),
    (16, 4200, 4, 2, 256, 4, 8),
    (1, 3000, 1, 2, 64, 16, 2),
    (1, 9000, 2, 5, 24, 16, 8),
    (1, 20000, 1, 2, 40, 16, 19),
    (1, 20000, 2, 8, 64, 16, 19),
    (2, 3000, 1, 3, 72, 8, 5),
    (1, 9000, 2, 4, 72, 8, 17),
    (1, 9000, 2, 2, 128, 8, 17),
    (1, 9000, 2, 1, 136, 8, 17),
    (1, 3000, 2, 6, 200, 8, 5),
    (1, 9000, 2, 2, 256, 8, 17),
]


@pytest.mark.parametrize(("b", "w", "hkv", "group", "dk", "waves", "splits"), FORMS)
def test_the_cases_reach_the_forms_they_name(b, w, hkv, group, dk, waves, splits):
    """On the CPU: the splits as the workspace's size tells them, the waves by the rule above."""
    from vesper.kernels import _lib

    nbytes = _lib.library().vsp_quant_ring_attn_workspace_bytes(b, hkv * group, hkv, dk, w)
    assert nbytes == (0 if splits == 1 else 4 * b * hkv * group * splits * (2 + dk))
    heads, runs = b * hkv, (w + 31) // 32 // (32 if dk <= 64 else 16)
    many = heads >= 256 or heads * min(max(runs, 1), 256) >= 512
    assert waves == (4 if many else 16 if dk <= 64 else 8)


def _rows(g, *shape, dtype):
    x = torch.randn(*shape, generator=g, device=GPU) + 0.5 * torch.randn(shape[-1], generator=g, device=GPU)
    return x.to(dtype)


def _filled(b, w, hkv, group, dk, dtype, seed, fill=None):
    """A ring that each row has gone round a little further than once (or filled up to ``fill`` tokens), the new token."""
    from vesper.kernels.ring_quant import quant_ring_empty, quant_ring_write

    g = torch.Generator(device=GPU).manual_seed(seed)
    n = w + 37 if fill is None else fill
    seen = torch.randint(w, n + 1, (b, 1), generator=g, device=GPU) if fill is None else torch.full((b, 1), n, device=GPU)
    k, v = _rows(g, b, n, hkv, dk, dtype=dtype), _rows(g, b, n, hkv, dk, dtype=dtype)
    ring = quant_ring_write(k, v, torch.arange(n, device=GPU).expand(b, n), quant_ring_empty(b, hkv, dk, w, dtype, GPU),
                            lengths=seen[:, 0])
    q = torch.randn(b, 1, hkv * group, dk, generator=g, device=GPU).to(dtype)
    return q, _rows(g, b, 1, hkv, dk, dtype=dtype), _rows(g, b, 1, hkv, dk, dtype=dtype), seen, ring


def _values(packed, pair):
    codes = torch.stack([packed % 16, packed // 16], -1).flatten(-2).double()
    return pair[..., 1:].double() + pair[..., :1].double() * codes


def _reference(q, k, v, pos, ring):
    """The attention in float64 on the GPU, all rows at once."""
    b, _, h, dk = q.shape
    hkv, w = k.shape[2], ring.window
    keys = torch.cat([_values(ring.k, ring.k_scale), k.transpose(1, 2).double()], 2)
    values = torch.cat([_values(ring.v, ring.v_scale), v.transpose(1, 2).double()], 2)
    slots = torch.arange(w, device=GPU)
    use = ring.valid & (ring.pos <= pos) & (ring.pos > pos - w) & (slots != pos % w)
    use = torch.cat([use, torch.ones_like(use[:, :1])], 1)[:, None, :, None]
    qt = q.view(b, hkv, h // hkv, dk).transpose(2, 3).double().contiguous()
    scores = (torch.matmul(keys, qt) / math.sqrt(dk)).masked_fill(~use, -math.inf)
    weights = torch.softmax(scores, 2).transpose(2, 3).contiguous()
    return torch.matmul(weights, values).view(b, 1, h, dk)


def _bound(q, ring, v, ref, dtype):
    f = lambda t: float(t.double().abs().max())  # noqa: E731
    sk, sv = f(ring.k_scale[..., 0]), f(ring.v_scale[..., 0])
    top = max(f(v), f(ring.v_scale[..., 1]) + 15 * sv)
    es = 8 * 2.0**-24 * 143 * sk * float(q.double().abs().sum(-1).max()) / math.sqrt(q.shape[-1])
    return HALF_EPS[dtype] * ref.abs() + 2 * es * top + 143 * sv * 2.0**-16 + 2.0**-20


def _attend(*args, **kw):
    from vesper.kernels.ring_quant import quant_ring_attention

    return quant_ring_attention(*args, **kw)


def _check(q, k, v, pos, ring, dtype):
    ref = _reference(q, k, v, pos, ring)
    o, out = _attend(q, k, v, pos, ring)
    over = (o.double() - ref).abs() / _bound(q, ring, v, ref, dtype)
    assert bool((over <= 1).all()), float(over.max())
    return o, out


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("b", "w", "hkv", "group", "dk", "waves", "splits"), FORMS)
def test_attention_in_every_form(b, w, hkv, group, dk, waves, splits, dtype):
    from vesper.kernels.ring_quant import quant_ring_write

    q, k, v, pos, ring = _filled(b, w, hkv, group, dk, dtype, seed=w + dk)
    o, out = _check(q, k, v, pos, ring, dtype)
    for mine, theirs in zip(out.tensors(), quant_ring_write(k, v, pos, ring).tensors()):
        assert torch.equal(mine, theirs)
    again, _ = _attend(q, k, v, pos, out)  # on the ring it wrote: the same slots are seen
    assert torch.equal(again, o)


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("b", "w", "hkv", "group", "dk", "fill"), [
    (32, 520, 8, 2, 64, 65), (16, 8191, 4, 3, 64, 1030), (8, 8300, 4, 2, 72, 2050), (1, 20000, 2, 8, 64, 19000), (1, 9000, 2, 2, 136, 33),
])
def test_rings_that_are_filled_in_part(b, w, hkv, group, dk, fill, dtype):
    """Waves, tiles and whole splits that see nothing beside ones that do."""
    q, k, v, pos, ring = _filled(b, w, hkv, group, dk, dtype, seed=fill, fill=fill)
    _check(q, k, v, pos, ring, dtype)


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize(("b", "w", "hkv", "dk"), [(1, 3000, 1, 64), (1, 20000, 1, 64), (8, 8300, 4, 72)])
def test_a_captured_step_over_a_split_window(b, w, hkv, dk):
    """Two, 19 and 16 splits: replays at advancing positions, eager calls of the same shape between them."""
    from vesper.kernels.ring_quant import QuantRingKVCache

    q, k, v, pos, ring = _filled(b, w, hkv, 2, dk, BF16, seed=w)
    clone = lambda r: QuantRingKVCache(*(t.clone() for t in r.tensors()), r.window)  # noqa: E731
    mine, check = clone(ring), clone(ring)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _attend(q, k, v, pos, clone(ring), inplace=True, check_positions=False)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, _ = _attend(q, k, v, pos, mine, inplace=True, check_positions=False)
    for t in range(4):
        graph.replay()
        want, _ = _attend(q, k, v, pos, check, inplace=True)
        torch.cuda.synchronize()
        assert torch.equal(o, want)
        for x, y in zip(mine.tensors(), check.tensors()):
            assert torch.equal(x, y)
        pos.add_(1)
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(t)).to(BF16))


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize(("b", "w", "hkv", "dk"), [(2, 70, 2, 64), (1, 3000, 2, 72)])
def test_the_c_entry_without_a_write(b, w, hkv, dk):
    """``write`` = 0: the same output, the ring as it was."""
    from vesper.kernels import _lib

    q, k, v, pos, ring = _filled(b, w, hkv, 2, dk, BF16, seed=dk)
    want, _ = _attend(q, k, v, pos, ring)
    before = [t.clone() for t in ring.tensors()]
    o = torch.full_like(q, math.nan)
    nbytes = _lib.library().vsp_quant_ring_attn_workspace_bytes(b, 2 * hkv, hkv, dk, w)
    room = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=GPU)
    _lib.call("vsp_quant_ring_attn_bf16", q.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(),
              *(t.data_ptr() for t in ring.tensors()), o.data_ptr(), None, room.data_ptr(), nbytes, b, 2 * hkv, hkv, dk, w,
              1.0 / math.sqrt(dk), 0, _lib.stream_of(q.device))
    assert torch.equal(o, want)
    for mine, old in zip(ring.tensors(), before):
        assert torch.equal(mine, old)


def _ring_of(k, v, w, dtype, after=0):
    """A ring of tokens ``k, v [b, n, hkv, dk]`` at positions 0 .. n - 1, and the position behind them."""
    from vesper.kernels.ring_quant import quant_ring_empty, quant_ring_write

    b, n, hkv, dk = k.shape
    k, v = k.to(dtype).to(GPU), v.to(dtype).to(GPU)
    ring = quant_ring_write(k, v, torch.arange(n, device=GPU).expand(b, n), quant_ring_empty(b, hkv, dk, w, dtype, GPU))
    return ring, torch.full((b, 1), n + after, device=GPU)


EDGES = [(1, 40, 1, 64), (2, 520, 2, 72), (1, 5000, 2, 64), (32, 260, 8, 128), (8, 8300, 4, 72), (1, 9000, 1, 136)]


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("size", [2.0**60, 2.0**100, 2.0**116, 2.0**120, 2.0**127])
@pytest.mark.parametrize(("b", "w", "hkv", "dk"), EDGES)
def test_values_up_to_the_largest_bf16_are_averaged(b, w, hkv, dk, size):
    """Every score 0, so that each weight is 1 and the sums are as many times the values as there are tokens."""
    g = torch.Generator().manual_seed(w)
    v = (2 * torch.rand(b, w, hkv, dk, generator=g, dtype=torch.float64) - 1) * size
    ring, pos = _ring_of(torch.randn(b, w, hkv, dk, generator=g), v, w, BF16)
    q = torch.zeros(b, 1, 2 * hkv, dk, dtype=BF16, device=GPU)
    _check(q, v[:, :1].to(BF16).to(GPU), v[:, 1:2].to(BF16).to(GPU), pos, ring, BF16)


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("gap", [0.0, 3.0, 400.0, 2.0**27])
@pytest.mark.parametrize("late", [False, True])
@pytest.mark.parametrize(("b", "w", "hkv", "dk"), EDGES)
def test_a_few_values_near_the_largest_among_small_ones(b, w, hkv, dk, late, gap):
    """Seven tokens in a row of 2^126 among ones of about 1, their scores ``gap`` lower (from 400 on they weigh
    nothing and the small ones are averaged as if alone), in the first tiles and in the last."""
    g = torch.Generator().manual_seed(w + dk)
    k, v = torch.zeros(b, w, hkv, dk), torch.randn(b, w, hkv, dk, generator=g, dtype=torch.float64)
    at = slice(w - 9, w - 2) if late else slice(2, 9)
    v[:, at] *= 2.0**126 / 4
    k[:, at, :, 0] = -gap
    ring, pos = _ring_of(k, v, w, BF16, after=1)
    q = torch.zeros(b, 1, hkv, dk, dtype=BF16, device=GPU)
    q[..., 0] = math.sqrt(dk)
    new_k, new_v = torch.zeros(b, 1, hkv, dk, dtype=BF16, device=GPU), torch.randn(b, 1, hkv, dk, generator=g).to(BF16).to(GPU)
    ref, (o, _) = _reference(q, new_k, new_v, pos, ring), _attend(q, new_k, new_v, pos, ring)
    err = (o.double() - ref).abs()
    if gap >= 400:  # the small rows' scales are below 1, whatever the large ones' are
        small = ring.v_scale[..., 0].double()
        sv = float(small[small < 2.0**60].max())
        assert bool((err <= HALF_EPS[BF16] * ref.abs() + 143 * sv * 2.0**-16 + 2.0**-20).all()), float(err.max())
    else:
        assert bool((err <= _bound(q, ring, new_v, ref, BF16)).all()), float(err.max())


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("size", [2.0**60, 2.0**116, 2.0**124, 2.0**127])
@pytest.mark.parametrize(("b", "w", "hkv", "dk"), EDGES)
def test_keys_up_to_the_largest_bf16_are_scored(b, w, hkv, dk, size):
    """Queries as small as the keys are large, so that the scores are of the usual size; and queries of 0, whose scores
    are 0 whatever the keys."""
    g = torch.Generator().manual_seed(w)
    k = (2 * torch.rand(b, w, hkv, dk, generator=g, dtype=torch.float64) - 1) * size
    ring, pos = _ring_of(k, torch.randn(b, w, hkv, dk, generator=g), w, BF16)
    new_v = torch.randn(b, 1, hkv, dk, generator=g).to(BF16).to(GPU)
    small = torch.randn(b, 1, 2 * hkv, dk, generator=g, dtype=torch.float64)
    small = (small.sign() * small.abs().clamp_min(0.5) / size * 2).to(BF16).to(GPU)  # no subnormal numbers
    for q in (small, torch.zeros_like(small)):
        _check(q, k[:, :1].to(BF16).to(GPU), new_v, pos, ring, BF16)


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("b", "w", "hkv", "dk"), EDGES)
def test_an_average_of_values_at_the_types_end_stays_in_the_type(b, w, hkv, dk, dtype):
    """Rows from -top to top: the scale's rounding takes the last code past the type's range, and the output, an average
    of numbers of the type, is brought back to its largest as the read brings back a value."""
    from vesper.kernels.ring_quant import quant_ring_read

    top = torch.finfo(dtype).max
    row = torch.linspace(-1, 1, dk, dtype=torch.float64) * top
    v = row.expand(b, w, hkv, dk).clone()
    ring, pos = _ring_of(torch.randn(b, w, hkv, dk), v, w, dtype)
    _, read, _ = quant_ring_read(ring, torch.zeros(b, 1, dtype=torch.long, device=GPU))
    q, new_k = torch.zeros(b, 1, hkv, dk, dtype=dtype, device=GPU), torch.zeros(b, 1, hkv, dk, dtype=dtype, device=GPU)
    for new_v in (read, read.flip(3)):  # the same values again, and others
        ref = _reference(q, new_k, new_v, pos, ring).clamp(-top, top)
        o, _ = _attend(q, new_k, new_v, pos, ring)
        assert bool(torch.isfinite(o).all())
        assert bool(((o.double() - ref).abs() <= _bound(q, ring, new_v, ref, dtype)).all())
    new_v = read.clone()
    new_v[..., 3] = math.inf  # an infinity is not brought back
    o, _ = _attend(q, new_k, new_v, pos, ring)
    assert bool((o[..., 3] == math.inf).all()) and bool(torch.isfinite(o[..., :3]).all())


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("w", [40, 5000])
def test_a_lone_score_of_minus_infinity_is_nan(w):
    """0 / 0 in the average: NaN, as a softmax over that score alone is."""
    from vesper.kernels.ring_quant import quant_ring_empty

    q, k = torch.ones(1, 1, 1, 64, dtype=BF16, device=GPU), torch.zeros(1, 1, 1, 64, dtype=BF16, device=GPU)
    k[..., 5] = -math.inf
    o, _ = _attend(q, k, torch.ones_like(k), torch.zeros(1, 1, dtype=torch.long, device=GPU),
                   quant_ring_empty(1, 1, 64, w, BF16, GPU))
    assert bool(o.isnan().all())


@pytest.mark.gpu
@needs_gpu
def test_a_captured_write_and_read_replay_as_the_eager_ones():
    """A padded batch, its positions and lengths checked in the graph, and a read of them: replays with other tokens,
    positions and lengths, eager calls of the same shapes between them."""
    from vesper.kernels.ring_quant import QuantRingKVCache, quant_ring_empty, quant_ring_read, quant_ring_write

    b, n, w, hkv, dk = 3, 5000, 1200, 2, 40
    g = torch.Generator(device=GPU).manual_seed(41)
    k, v = _rows(g, b, n, hkv, dk, dtype=BF16), _rows(g, b, n, hkv, dk, dtype=BF16)
    pos, lengths = torch.arange(n, device=GPU).expand(b, n).contiguous(), torch.tensor([n, 0, 700], device=GPU)
    mine, check = quant_ring_empty(b, hkv, dk, w, BF16, GPU), quant_ring_empty(b, hkv, dk, w, BF16, GPU)
    run = lambda ring: (quant_ring_write(k, v, pos, ring, lengths=lengths, inplace=True), quant_ring_read(ring, pos[:, ::7]))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(QuantRingKVCache(*(t.clone() for t in mine.tensors()), w))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, got = run(mine)
    for t in range(4):
        graph.replay()
        _, want = run(check)
        torch.cuda.synchronize()
        for x, y in zip((*got, *mine.tensors()), (*want, *check.tensors())):
            assert torch.equal(x, y)
        pos.add_(lengths[:, None])
        k.copy_(_rows(g, b, n, hkv, dk, dtype=BF16))
        lengths.copy_(torch.tensor([17 * t, n - t, 1250], device=GPU))


@pytest.mark.gpu
@needs_gpu
def test_the_longest_window():
    """2^29 - 64 slots of one head of eight (2 GiB of codes less a little; 4 GiB of positions), a chunk that wraps round
    the end: as a small ring of the same tokens, written, read back and attended."""
    from vesper.kernels.ring_quant import quant_ring_empty, quant_ring_read, quant_ring_write

    w, n, dk = 2**29 - 64, 90, 8
    if torch.cuda.mem_get_info()[0] < 40 * 2**30:
        pytest.skip("needs 40 GiB of free GPU memory")
    g = torch.Generator(device=GPU).manual_seed(50)
    k, v = _rows(g, 1, n, 1, dk, dtype=BF16), _rows(g, 1, n, 1, dk, dtype=BF16)
    start = 9 * w - 50
    pos = start + torch.arange(n, device=GPU)[None]
    ring = quant_ring_write(k, v, pos, quant_ring_empty(1, 1, dk, w, BF16, GPU), inplace=True)
    small = quant_ring_write(k, v, pos - start, quant_ring_empty(1, 1, dk, 128, BF16, GPU))
    for a, b in zip(quant_ring_read(ring, pos), quant_ring_read(small, pos - start)):
        assert torch.equal(a, b)
    assert int(ring.valid.sum()) == n and bool(ring.valid[0, -50:].all()) and bool(ring.valid[0, :n - 50].all())
    q = torch.randn(1, 1, 4, dk, generator=g, device=GPU).to(BF16)
    nk, nv = _rows(g, 1, 1, 1, dk, dtype=BF16), _rows(g, 1, 1, 1, dk, dtype=BF16)
    at = pos[:, -1:] + 1
    ref = _reference(q, nk, nv, at - start, small)
    o, _ = _attend(q, nk, nv, at, ring, inplace=True)
    assert bool(((o.double() - ref).abs() <= _bound(q, small, nv, ref, BF16)).all())
    assert int(ring.pos[0, n - 50]) == int(at) and int(ring.valid.sum()) == n + 1
    del ring
    torch.cuda.empty_cache()
