"""The sizes that the gated scan and step take, on the CPU, with tensors that have sizes and no memory."""

from __future__ import annotations

import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32


class _Wide(torch.Tensor):
    """One element seen as any shape, that says it lies on a GPU (one that no machine has, so that no kernel is reached)."""

    @property
    def device(self):
        return torch.device("cuda", 99)


def _of(*shape, dtype=F32):
    return torch.zeros(1, dtype=dtype).expand(*shape).as_subclass(_Wide)


def _args(b, n, h, dk, dtype=BF16):
    lead = (b, h) if n is None else (b, n, h)
    return [*(_of(*lead, dk, dtype=dtype) for _ in range(3)), _of(*lead, dtype=dtype), _of(*lead), _of(b, h, dk, dk)]


@pytest.fixture
def reached(monkeypatch):
    """What would be launched: ``(entry, arguments)`` of each call, in place of the launches."""
    from vesper.kernels import _lib

    calls = []
    monkeypatch.setattr(_lib, "launch", lambda device, name, *args: calls.append((name, args)))
    return calls


SCANS = [((1, 2**30 + 1, 1, 8), "tokens a row"), ((1, 2**32 + 8, 1, 8), "tokens a row"), ((1, 2, 2**20, 8), "features a token"),
         ((1, 2, 2**19, 9), "features a token"), ((2**25, 65, 1, 8), "chunks"), ((2**13, 2**18 + 1, 1, 8), "chunks"),
         ((2**22 + 1, 2, 1, 8), "slices"), ((2**20, 2, 2, 40), "slices"), ((2**33, 2, 1, 8), "chunks")]


@pytest.mark.parametrize(("size", "text"), SCANS, ids=str)
def test_scans_past_the_limits_are_refused(reached, size, text):
    from vesper.contracts import ContractError
    from vesper.kernels.gated_scan import gated_delta_scan

    with torch.no_grad(), pytest.raises(ContractError, match=text):
        gated_delta_scan(*_args(*size))
    assert not reached


def test_a_scan_that_keeps_records_takes_fewer_chunks(reached):
    """Its backward has 512 threads a chunk: 2^23 of them are 2^32."""
    from vesper.contracts import ContractError
    from vesper.kernels.gated_scan import gated_delta_scan

    args = _args(2**12, 2**17, 1, 8)
    with pytest.raises(ContractError, match="2\\*\\*23"):
        gated_delta_scan(*args[:4], args[4].detach().requires_grad_(), args[5])
    assert not reached


@pytest.mark.parametrize("size", [(1, 2**30, 1, 256, False), (1, 2**29 - 64, 1, 256, True), (1, 64, 2**19, 1, False), (1, 64, 2**14, 256, False), (2**25 // 8, 512, 1, 8, False),
                                  (2**22, 64, 1, 16, True), (2**23 - 1, 64, 1, 16, True)], ids=str)
def test_the_limits_themselves_are_taken(size):
    from vesper.contracts import ContractError
    from vesper.kernels.gated_scan import _check_sizes

    if size[0] == 2**23 - 1:  # as many chunks as the backward takes, but more slices
        with pytest.raises(ContractError, match="slices"):
            _check_sizes(*size)
    else:
        _check_sizes(*size)


def test_the_records_are_of_whole_tiles():
    from vesper.kernels import _lib

    lib = _lib.library()
    for dk, wide in ((8, 16), (16, 16), (24, 32), (40, 48), (136, 144), (256, 256)):
        assert lib.vsp_gated_scan_records_bytes(3, 70, 5, dk) == 3 * 5 * 2 * 4 * wide * (wide + 64)


def test_the_c_entries_refuse_as_many_chunks():
    from vesper.kernels import _lib

    lib = _lib.library()
    sizes = (2**12, 2**17, 1, 8)
    assert lib.vsp_gated_scan_backward_bf16(*[None] * 6, 0, *[None] * 10, 0, *sizes, None) != 0
    assert "2^23" in lib.vsp_last_error().decode()
    assert lib.vsp_gated_scan_f32(*[None] * 9, 0, 16, 0, None, *sizes, None) != 0  # with records
    assert "2^23" in lib.vsp_last_error().decode()
    assert lib.vsp_gated_scan_f32(*[None] * 9, 0, None, 0, None, *sizes, None) != 0  # without
    assert "null" in lib.vsp_last_error().decode()
    assert lib.vsp_gated_scan_backward_bf16(*[None] * 6, 0, *[None] * 10, 0, 2**12, 2**17 - 64, 1, 8, None) != 0
    assert "null" in lib.vsp_last_error().decode()


def test_a_step_of_more_heads_than_a_launch_takes_runs_in_parts(reached):
    """2^20 heads and more, by the step and by a scan of one token: rows of fewer than 2^20 heads a launch, in order."""
    from vesper.kernels.gated_scan import gated_delta_scan, gated_delta_step

    b, h, dk = 2**17 + 3, 8, 1
    lead = [torch.zeros(b, h, dk, dtype=BF16).as_subclass(_Wide) for _ in range(3)]
    beta, g = torch.zeros(b, h, dtype=BF16).as_subclass(_Wide), torch.zeros(b, h).as_subclass(_Wide)
    state = torch.zeros(b, h, dk, dk).as_subclass(_Wide)
    active = torch.ones(b, dtype=torch.bool).as_subclass(_Wide)
    with torch.no_grad():
        o, after = gated_delta_step(*lead, beta, g, state, active=active, out_state=state)
        assert o.shape == (b, h, dk) and after is state
        gated_delta_scan(*(t[:, None] for t in lead), beta[:, None], g[:, None], state)
    assert len(reached) == 4 and {name for name, _ in reached} == {"vsp_gated_step_bf16"}
    for calls in (reached[:2], reached[2:]):
        first = 0
        for _, args in calls:
            rows, heads, width = args[-3:]
            assert rows * heads < 2**20 and (heads, width) == (h, dk)
            for at, t in zip(args, (*lead, beta, g, state)):
                assert at == t.data_ptr() + first * t[:1].nbytes
            first += rows
        assert first == b
    first = reached[0][1][-3]
    for before, behind, t in zip(reached[0][1][6:9], reached[1][1][6:9], (state, o, active)):
        assert before == t.data_ptr() and behind == t.data_ptr() + first * t[:1].nbytes


def test_a_step_of_more_heads_a_row_is_refused(reached):
    from vesper.contracts import ContractError
    from vesper.kernels.gated_scan import gated_delta_step

    with pytest.raises(ContractError, match="heads"):
        gated_delta_step(*_args(1, None, 2**20, 1))
    assert not reached


@pytest.mark.parametrize("which", range(5))
def test_a_new_state_over_another_input_is_refused(reached, which):
    """Tokens within or at the ends of out_state's memory; right before and right behind it they are taken."""
    from vesper.contracts import ContractError
    from vesper.kernels.gated_scan import gated_delta_step

    b, h, dk = 2, 3, 4
    sizes = [b * h * dk] * 3 + [b * h] * 2
    shapes = [(b, h, dk)] * 3 + [(b, h)] * 2
    buf = torch.zeros(1000)
    held = buf[300 : 300 + b * h * dk * dk]
    out = held.view(b, h, dk, dk).as_subclass(_Wide)
    tokens = [torch.zeros(s).as_subclass(_Wide) for s in shapes]
    size = sizes[which]

    def call(at, **more):
        args = list(tokens)
        args[which] = buf[at : at + size].view(shapes[which]).as_subclass(_Wide)
        return gated_delta_step(*args, **more)

    for state in (out, torch.zeros(b, h, dk, dk).as_subclass(_Wide)):
        for at in (300 - size + 1, 300, 310, 300 + held.numel() - 1):
            with pytest.raises(ContractError, match="overlap"):
                call(at, state=state, out_state=out)
        for at in (300 - size, 300 + held.numel()):
            call(at, state=state, out_state=out)
    call(310, state=out)  # read only
    assert len(reached) == 5
