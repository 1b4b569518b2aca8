"""The gated delta rule's kernels against the float64 oracle: scan, gradients, step, and what can go wrong around them.

Tolerances, relative to the 2-norm of what is compared. A result held in bfloat16 is off by at most half a step of
each value, 2^-8; the products before it add sums of at most 256 + 64 terms in float32, 320 * 2^-24 = 1.9e-5 of the
magnitudes summed, and the outputs' operands of two bf16 pieces 2^-17 each: 2^-8 + 1e-4 in all. What is held in
float32 has the sums alone, three after each other a chunk: 3 * 1.9e-5 = 6e-5. The rounding errors are random, so
that what is seen is far below (about 2e-3 and 3e-7).
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import needs_gpu
from oracle.gated import gated_scan, gated_step

pytestmark = [pytest.mark.gpu, needs_gpu]

GPU = torch.device("cuda")
BF16, F32 = torch.bfloat16, torch.float32
HELD16, HELD32 = 2.0**-8 + 1e-4, 6e-5
NAMES = ("q", "k", "v", "beta", "g", "state")


def _inputs(b, n, h, dk, dtype, seed=0, resets=False, lead=None):
    gen = torch.Generator().manual_seed(seed)
    lead = (b, n, h) if lead is None else lead
    q, k, v = (torch.randn(*lead, dk, generator=gen) for _ in range(3))
    k = k + 0.4 * torch.randn(h, dk, generator=gen)
    k = k / k.norm(dim=-1, keepdim=True)
    beta = torch.sigmoid(torch.randn(*lead, generator=gen))
    rate = torch.exp(torch.linspace(math.log(1e-3), math.log(2.0), h))
    g = -rate * torch.nn.functional.softplus(torch.randn(*lead, generator=gen))
    if resets:
        g = torch.where(torch.rand(*lead[:2], 1, generator=gen) < 0.02, torch.full_like(g, -math.inf), g)
    state = 0.5 * torch.randn(b, h, dk, dk, generator=gen)
    return [q.to(GPU, dtype), k.to(GPU, dtype), v.to(GPU, dtype), beta.to(GPU, dtype), g.to(GPU), state.to(GPU)]


def _oracle(inputs, active=None):
    o, after = gated_scan(*(t.detach().cpu().double() for t in inputs), None if active is None else active.cpu())
    return o, after


def _close(got, want, held=None, what=""):
    held = (HELD16 if got.dtype == BF16 else HELD32) if held is None else held
    got, want = got.detach().cpu().double(), want.detach().cpu().double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    off = float((got - want).norm())
    assert off <= held * float(want.norm()) + 1e-30, (what, off / max(float(want.norm()), 1e-30))


SIZES = [(1, 1, 1, 8), (2, 2, 1, 8), (1, 63, 2, 16), (2, 64, 1, 24), (1, 65, 3, 32), (3, 17, 5, 64), (2, 129, 2, 64),
         (1, 130, 2, 72), (1, 100, 2, 128), (1, 200, 1, 136), (1, 70, 1, 256), (1, 80, 3, 20), (2, 66, 2, 1), (1, 90, 1, 255)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("resets", [False, True])
def test_scan_matches_the_oracle(dtype, size, resets):
    from vesper.kernels.gated_scan import gated_delta_scan

    inputs = _inputs(*size, dtype, seed=sum(size), resets=resets)
    with torch.no_grad():
        o, after = gated_delta_scan(*inputs)
    want, last = _oracle(inputs)
    assert o.dtype == dtype and after.dtype == F32
    _close(o, want, what="o")
    _close(after, last, what="state")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("masked", [False, True])
def test_gradients_match_the_oracle(dtype, size, masked):
    from vesper.kernels.gated_scan import gated_delta_scan

    b, n, h, dk = size
    inputs = _inputs(*size, dtype, seed=sum(size) + 1, resets=masked)
    gen = torch.Generator().manual_seed(7)
    do, ds = torch.randn(b, n, h, dk, generator=gen).to(GPU, dtype), torch.randn(b, h, dk, dk, generator=gen).to(GPU)
    active = (torch.rand(b, n, generator=gen) < 0.7).to(GPU) if masked else None
    leaves = [t.requires_grad_() for t in inputs]
    o, after = gated_delta_scan(*leaves, active=active)
    got = torch.autograd.grad([o, after], leaves, [do, ds])
    exact = [t.detach().cpu().double().requires_grad_() for t in inputs]
    want_o, want_after = gated_scan(*exact, None if active is None else active.cpu())
    want = torch.autograd.grad([want_o, want_after], exact, [do.cpu().double(), ds.cpu().double()])
    _close(o, want_o, what="o")
    _close(after, want_after, what="state")
    if active is not None:
        assert not bool(o[~active].any())
    for name, x, y, t in zip(NAMES, got, want, inputs):
        assert x.dtype == t.dtype
        _close(x, torch.nan_to_num(y), what=name)
    if masked:
        assert not bool(got[4][torch.isinf(inputs[4])].any())  # what forgets has no gradient


def test_gradients_against_differences():
    """The directional derivative of the float64 oracle by central differences against the kernels' gradients: steps of
    1e-4 are off by about 1e-8 of the third derivative, far below the float32 gradients' 6e-5."""
    from vesper.kernels.gated_scan import gated_delta_scan

    inputs = _inputs(1, 70, 2, 16, F32, seed=5)
    gen = torch.Generator().manual_seed(1)
    do, ds = torch.randn(1, 70, 2, 16, generator=gen), torch.randn(1, 2, 16, 16, generator=gen)
    leaves = [t.requires_grad_() for t in inputs]
    grads = torch.autograd.grad(list(gated_delta_scan(*leaves)), leaves, [do.to(GPU), ds.to(GPU)])
    exact = [t.detach().cpu().double() for t in inputs]

    def loss(args):
        o, after = gated_scan(*args)
        return float((o * do.double()).sum() + (after * ds.double()).sum())

    for i, name in enumerate(NAMES):
        way = torch.randn(exact[i].shape, generator=gen, dtype=torch.float64)
        near = [loss([t + (s * 1e-4 * way if j == i else 0) for j, t in enumerate(exact)]) for s in (1, -1)]
        want = (near[0] - near[1]) / 2e-4
        got = float((grads[i].cpu().double() * way).sum())
        scale = float(grads[i].cpu().double().norm() * way.norm())
        assert abs(got - want) <= (HELD32 + 1e-6) * scale, name


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_only_one_of_the_results_is_used(dtype):
    from vesper.kernels.gated_scan import gated_delta_scan

    for which in (0, 1):
        leaves = [t.requires_grad_() for t in _inputs(2, 100, 2, 32, dtype, seed=3)]
        got = torch.autograd.grad(gated_delta_scan(*leaves)[which].float().sin().sum(), leaves, allow_unused=True)
        exact = [t.detach().cpu().double().requires_grad_() for t in leaves]
        want = torch.autograd.grad(gated_scan(*exact)[which].sin().sum(), exact, allow_unused=True)
        for name, x, y in zip(NAMES, got, want):
            y = torch.zeros_like(x, device="cpu", dtype=torch.float64) if y is None else y
            # the loss's own gradient is of rounded outputs: 2^-8 of their values, of slope at most one
            _close(x, y, held=3 * HELD16 if dtype == BF16 else HELD32, what=name)


def test_a_second_derivative_is_refused():
    from vesper.kernels.gated_scan import gated_delta_scan

    leaves = [t.requires_grad_() for t in _inputs(1, 5, 1, 8, F32)]
    first = torch.autograd.grad(gated_delta_scan(*leaves)[0].square().sum(), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first[0].sum().backward()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_without_decay_it_is_the_delta_scan(dtype):
    from vesper.kernels.delta_scan import delta_scan_fused, delta_scan_fused_fp32
    from vesper.kernels.gated_scan import gated_delta_scan

    q, k, v, beta, g, state = _inputs(2, 200, 2, 64, dtype)
    with torch.no_grad():
        mine = gated_delta_scan(q, k, v, beta, torch.zeros_like(g), state)
        theirs = (delta_scan_fused if dtype == BF16 else delta_scan_fused_fp32)(q, k, v, beta, state)
    for a, b in zip(mine, theirs):
        _close(a, b, held=1.5e-2 if dtype == BF16 else 1e-5)  # the delta scan's own tolerances


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_block_in_parts_is_the_block(dtype):
    """Parts that start anew within a chunk: the same sums in another order."""
    from vesper.kernels.gated_scan import gated_delta_scan

    *tokens, state = _inputs(2, 300, 3, 40, dtype, seed=9, resets=True)
    with torch.no_grad():
        whole, after = gated_delta_scan(*tokens, state)
        outs = []
        for s, e in ((0, 1), (1, 70), (70, 71), (71, 200), (200, 300)):
            o, state = gated_delta_scan(*(t[:, s:e] for t in tokens), state)
            outs.append(o)
    _close(torch.cat(outs, 1), whole, held=2 * HELD16 if dtype == BF16 else 2 * HELD32)
    _close(state, after, held=2 * HELD32)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize(("b", "h", "dk"), [(1, 1, 1), (3, 2, 7), (2, 3, 16), (1, 2, 33), (5, 8, 64), (2, 2, 96), (1, 1, 130),
                                            (1, 2, 255), (1, 2, 256), (64, 8, 64), (300, 3, 128)])
@pytest.mark.parametrize("inplace", [False, True])
def test_step_matches_the_oracle(dtype, b, h, dk, inplace):
    from vesper.kernels.gated_scan import gated_delta_step

    inputs = _inputs(b, 1, h, dk, dtype, seed=b + dk, lead=(b, h))
    inputs[4][0] = -math.inf  # forgets
    active = torch.arange(b, device=GPU) % 3 != 1
    want, after = gated_step(*(t.cpu().double() for t in inputs))
    before = inputs[5].clone()
    o, new = gated_delta_step(*inputs, active=active, out_state=inputs[5] if inplace else None)
    assert (new is inputs[5]) == inplace and (inplace or torch.equal(inputs[5], before))
    _close(o, want * active.cpu()[:, None, None])
    assert not bool(o[~active].any())
    _close(new, after)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_steps_are_the_scan(dtype):
    from vesper.kernels.gated_scan import gated_delta_scan, gated_delta_step

    *tokens, state = _inputs(2, 70, 2, 64, dtype, seed=4)
    with torch.no_grad():
        whole, after = gated_delta_scan(*tokens, state)
        one, first = gated_delta_scan(*(t[:, :1] for t in tokens), state)  # one token of a scan is a step
        outs = []
        for t in range(70):
            o, state = gated_delta_step(*(x[:, t] for x in tokens), state.contiguous())
            if t == 0:
                assert torch.equal(o, one[:, 0]) and torch.equal(state, first)
            outs.append(o)
    _close(torch.stack(outs, 1), whole, held=2 * HELD16 if dtype == BF16 else 2 * HELD32)
    _close(state, after, held=2 * HELD32)


def _strided(t):
    """The same values behind other strides and an odd offset."""
    order = list(range(t.dim()))[::-1]
    buf = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view([t.shape[i] for i in order])
    out = buf.permute(order)
    out.copy_(t)
    assert t.numel() == 1 or not out.is_contiguous()
    return out


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strided_and_unaligned_inputs_are_the_contiguous_ones(dtype):
    from vesper.kernels.gated_scan import gated_delta_scan, gated_delta_step

    inputs = _inputs(2, 67, 3, 24, dtype)
    do, ds = torch.randn_like(inputs[0]), torch.randn_like(inputs[5])
    results = []
    for change in (lambda t: t, _strided):
        leaves = [change(t).detach().requires_grad_() for t in inputs]
        o, after = gated_delta_scan(*leaves)
        results.append([o, after, *torch.autograd.grad([o, after], leaves, [change(do), change(ds)])])
        with torch.no_grad():
            results[-1] += gated_delta_step(*(change(t)[:, 0] for t in inputs[:5]), inputs[5])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_results_repeat_bit_for_bit_and_on_another_stream(dtype):
    from vesper.kernels.gated_scan import gated_delta_scan

    inputs = _inputs(3, 260, 4, 64, dtype, resets=True)
    do = torch.randn_like(inputs[0])
    side = torch.cuda.Stream()

    def once():
        leaves = [t.detach().requires_grad_() for t in inputs]
        o, after = gated_delta_scan(*leaves)
        return [o, after, *torch.autograd.grad([o, after], leaves, [do, after.detach()])]

    first, second = once(), once()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        third = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_captured_training_step_and_decode_step_replay_as_the_eager_ones(dtype):
    from vesper.kernels.gated_scan import gated_delta_scan, gated_delta_step

    b, n, h, dk = 2, 150, 2, 64
    held = [t.detach().requires_grad_() for t in _inputs(b, n, h, dk, dtype, seed=1)]
    do, ds = torch.randn(b, n, h, dk, device=GPU, dtype=dtype), torch.randn(b, h, dk, dk, device=GPU)
    decoding = torch.zeros(b, h, dk, dk, device=GPU)

    def work():
        o, after = gated_delta_scan(*held)
        grads = torch.autograd.grad([o, after], held, [do, ds])
        with torch.no_grad():
            read, _ = gated_delta_step(*(t.detach()[:, 0] for t in held[:5]), decoding, out_state=decoding)
        return [o.detach(), after.detach(), *grads, read]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = work()
    for seed in (2, 3, 4):
        fresh = _inputs(b, n, h, dk, dtype, seed=seed, resets=seed == 4)
        with torch.no_grad():
            for t, x in zip(held, fresh):
                t.copy_(x)
            decoding.copy_(fresh[5])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*static, decoding)]
        decoding.copy_(fresh[5])
        want = [*work(), decoding]
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y), seed


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["forgets", "keeps", "no keys", "no writes", "large", "small", "one key", "fast"])
def test_extremes(dtype, kind):
    from vesper.kernels.gated_scan import gated_delta_scan

    inputs = _inputs(1, 140, 2, 32, dtype, seed=11)
    q, k, v, beta, g, state = inputs
    if kind == "forgets":
        g.fill_(-math.inf)
    elif kind == "keeps":
        g.zero_()
    elif kind == "no keys":
        k.zero_()
    elif kind == "no writes":
        beta.zero_()
    elif kind in ("large", "small"):
        scale = 2.0**60 if kind == "large" else 2.0**-60
        v.mul_(scale)
        state.mul_(scale)
    elif kind == "one key":  # every token overwrites the last one's value: the inverse's longest chains
        k.copy_(k[:, :1].clone())
        beta.fill_(1.0)
        g.zero_()
    else:
        g.fill_(-300.0)  # sums of -19200 a chunk: differences that float32 sums would round by 1e-3
        g[:, ::3] = -1e-3
    leaves = [t.requires_grad_() for t in inputs]
    gen = torch.Generator().manual_seed(2)
    do, ds = torch.randn(q.shape, generator=gen).to(GPU, dtype), torch.randn(state.shape, generator=gen).to(GPU)
    o, after = gated_delta_scan(*leaves)
    got = [o, after, *torch.autograd.grad([o, after], leaves, [do, ds])]
    exact = [t.detach().cpu().double().requires_grad_() for t in inputs]
    o, after = gated_scan(*exact)
    want = [o, after, *torch.autograd.grad([o, after], exact, [do.cpu().double(), ds.cpu().double()])]
    for name, x, y in zip(("o", "after", *NAMES), got, want):
        y = torch.nan_to_num(y)  # 0 times the infinite decay's derivative
        if name == "g" and not float(y.norm()):
            assert float(x.norm()) == 0.0
            continue
        if name == "g" and kind == "fast":
            # gradients of decays of e^-300 are zeros beside sums of both signs: off by float32's rounding of those
            _close(x, y, held=1e-3, what=name)
            continue
        # states that hold one value of every 140 written come of differences of all of them
        _close(x, y, held=4 * HELD32 if kind == "one key" and x.dtype == F32 else None, what=name)


@pytest.mark.parametrize("token", [50, 80])
def test_a_nan_stays_in_its_head_and_row(token):
    """And behind the start of its chunk of 64 tokens: within it, the products over all pairs of tokens meet it."""
    from vesper.kernels.gated_scan import gated_delta_scan

    inputs = _inputs(2, 100, 3, 64, BF16, seed=6)
    clean = [t.clone() for t in inputs]
    inputs[2][0, token, 1, 5] = math.nan
    do = torch.randn_like(inputs[0])
    runs = []
    for args in (inputs, clean):
        leaves = [t.requires_grad_() for t in args]
        o, after = gated_delta_scan(*leaves)
        runs.append([o, after, *torch.autograd.grad([o, after], leaves, [do, torch.ones_like(after)])])
    for name, x, y in zip(("o", "after", *NAMES), *runs):
        head = 1 if name in ("after", "state") else 2
        keep = torch.ones(x.shape[0], x.shape[head], dtype=torch.bool, device=GPU)
        keep[0, 1] = False
        x, y = (t.movedim(head, 1)[keep] for t in (x, y))
        assert torch.equal(x, y), name
    assert bool(torch.isnan(runs[0][0][0, token:, 1]).any())
    start = token // 64 * 64
    assert torch.equal(runs[0][0][0, :start, 1], runs[1][0][0, :start, 1])


def test_empty_batches():
    from vesper.kernels.gated_scan import gated_delta_scan, gated_delta_step

    for b, h in ((0, 2), (2, 0)):
        args = [torch.zeros(b, 5, h, 16, device=GPU, dtype=BF16)] * 3 + [torch.zeros(b, 5, h, device=GPU, dtype=BF16),
                torch.zeros(b, 5, h, device=GPU), torch.zeros(b, h, 16, 16, device=GPU)]
        o, after = gated_delta_scan(*args)
        assert o.shape == args[0].shape and after.shape == args[5].shape
        o, after = gated_delta_step(*(t[:, 0] for t in args[:5]), args[5])
        assert o.shape == (b, h, 16) and after.shape == args[5].shape


def test_offsets_past_32_bits():
    """The last row of a batch of more than 2^31 elements, and of more than 2^31 bytes of chunk records, is the row alone."""
    from vesper.kernels.gated_scan import gated_delta_scan

    b, n, h, dk = 33, 16448, 64, 64  # 2.2e9 elements
    gen = torch.Generator(device=GPU).manual_seed(0)
    q, k, v = (torch.empty(b, n, h, dk, device=GPU, dtype=BF16).normal_(generator=gen) for _ in range(3))
    k.mul_(0.1)
    beta = torch.rand(b, n, h, device=GPU, generator=gen).to(BF16)
    g = -torch.rand(b, n, h, device=GPU, generator=gen)
    state = torch.randn(b, h, dk, dk, device=GPU, generator=gen)
    with torch.no_grad():
        o, after = gated_delta_scan(q, k, v, beta, g, state)
        alone, last = gated_delta_scan(*(t[-1:] for t in (q, k, v, beta, g, state)))
    assert torch.equal(o[-1:], alone) and torch.equal(after[-1:], last)


# few long rows: the sequence in segments, whose starting states are joined first
LONG = [(1, 2100, 2, 64), (2, 2048, 1, 16), (1, 4095, 1, 64), (1, 2500, 1, 128), (1, 2049, 1, 200), (1, 2177, 3, 20)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", LONG, ids=str)
@pytest.mark.parametrize("resets", [False, True])
def test_long_rows_match_the_oracle(dtype, size, resets):
    from vesper.kernels.gated_scan import gated_delta_scan

    inputs = _inputs(*size, dtype, seed=sum(size), resets=resets)
    active = (torch.rand(*size[:2], generator=torch.Generator().manual_seed(3)) < 0.8).to(GPU) if resets else None
    with torch.no_grad():
        o, after = gated_delta_scan(*inputs, active=active)
    want, last = _oracle(inputs, active)
    _close(o, want, what="o")
    _close(after, last, what="state")
    if active is not None:
        assert not bool(o[~active].any())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [(1, 2100, 2, 64), (1, 2048, 1, 24)], ids=str)
def test_gradients_of_long_rows_match_the_oracle(dtype, size):
    from vesper.kernels.gated_scan import gated_delta_scan

    b, n, h, dk = size
    inputs = _inputs(*size, dtype, seed=sum(size))
    gen = torch.Generator().manual_seed(2)
    do, ds = torch.randn(b, n, h, dk, generator=gen).to(GPU, dtype), torch.randn(b, h, dk, dk, generator=gen).to(GPU)
    leaves = [t.requires_grad_() for t in inputs]
    o, after = gated_delta_scan(*leaves)
    got = torch.autograd.grad([o, after], leaves, [do, ds])
    exact = [t.detach().cpu().double().requires_grad_() for t in inputs]
    want_o, want_after = gated_scan(*exact)
    want = torch.autograd.grad([want_o, want_after], exact, [do.cpu().double(), ds.cpu().double()])
    _close(o, want_o, what="o")
    _close(after, want_after, what="state")
    for name, x, y in zip(NAMES, got, want):
        _close(x, y, what=name)
    with torch.no_grad():
        plain, last = gated_delta_scan(*(t.detach() for t in inputs))
    assert torch.equal(plain, o) and torch.equal(last, after)  # with and without records


def test_long_rows_keep_a_nan_to_its_head_and_what_follows():
    """Chunks before the one with the NaN, and the other head, are bit for bit as without it."""
    from vesper.kernels.gated_scan import gated_delta_scan

    inputs = _inputs(1, 2100, 2, 64, BF16, seed=9)
    with torch.no_grad():
        o, after = gated_delta_scan(*inputs)
        inputs[2][0, 1000, 1, 5] = math.nan  # token 1000: chunk 15, the tokens 960 .. 1023
        bad, bad_after = gated_delta_scan(*inputs)
    assert torch.equal(bad[:, :960], o[:, :960]) and torch.equal(bad[:, :, 0], o[:, :, 0])
    assert torch.equal(bad_after[:, 0], after[:, 0]) and bool(bad_after[0, 1].isnan().any())


def test_long_rows_in_a_graph():
    from vesper.kernels.gated_scan import gated_delta_scan

    inputs = _inputs(1, 2100, 2, 64, BF16, seed=4)
    side = torch.cuda.Stream()
    with torch.no_grad(), torch.cuda.stream(side):
        gated_delta_scan(*inputs)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            o, after = gated_delta_scan(*inputs)
    torch.cuda.synchronize()
    for seed in (5, 6, 7):
        for t, x in zip(inputs, _inputs(1, 2100, 2, 64, BF16, seed=seed)):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            want, last = gated_delta_scan(*inputs)
        assert torch.equal(o, want) and torch.equal(after, last)


# more chunks and heads than CUs: the other form of the chunks' factors
MANY = [(20, 200, 4, 64), (9, 70, 15, 32), (33, 130, 3, 16), (17, 65, 8, 128), (1, 70, 131, 136), (5, 64, 60, 8), (2, 5, 130, 256)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", MANY, ids=str)
@pytest.mark.parametrize("resets", [False, True])
def test_many_chunks_match_the_oracle(dtype, size, resets):
    test_scan_matches_the_oracle(dtype, size, resets)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [(20, 200, 4, 64), (33, 130, 3, 16), (17, 65, 8, 72), (9, 70, 15, 24)], ids=str)
@pytest.mark.parametrize("masked", [False, True])
def test_gradients_of_many_chunks_match_the_oracle(dtype, size, masked):
    test_gradients_match_the_oracle(dtype, size, masked)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dk", [32, 64, 128, 256])
def test_a_row_among_many_is_the_row_alone(dtype, dk):
    """Rows of a large batch (a wave a chunk in the first kernel) bit for bit as alone (four waves a chunk), gradients too."""
    from vesper.kernels.gated_scan import gated_delta_scan

    b, n, h = 90, 130, 1
    inputs = _inputs(b, n, h, dk, dtype, seed=dk, resets=True)
    do = torch.randn(b, n, h, dk, device=GPU, generator=torch.Generator(GPU).manual_seed(1)).to(dtype)
    leaves = [t.detach().requires_grad_() for t in inputs]
    o, after = gated_delta_scan(*leaves)
    grads = torch.autograd.grad([o, after], leaves, [do, torch.ones_like(after)])
    for row in (0, 41, 89):
        alone = [t[row : row + 1].detach().clone().requires_grad_() for t in inputs]
        o1, after1 = gated_delta_scan(*alone)
        grads1 = torch.autograd.grad([o1, after1], alone, [do[row : row + 1].clone(), torch.ones_like(after1)])
        for name, x, y in zip(("o", "state", *NAMES), (o, after, *grads), (o1, after1, *grads1)):
            assert torch.equal(x[row : row + 1], y), (name, row)
