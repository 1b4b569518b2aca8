"""What the few-bit operators refuse, on the CPU: shapes, dtypes, widths, devices and gradients, at the Python
boundary and at the C ABI, before any launch; and the float64 quantiser of the tests."""

from __future__ import annotations

import math

import pytest
import torch

BF16 = torch.bfloat16


def _ring(b=2, hkv=2, dk=16, w=8, dtype=BF16):
    from vesper.kernels.ring_quant import quant_ring_empty

    return quant_ring_empty(b, hkv, dk, w, dtype, torch.device("cpu"))


def _token(b=2, h=2, dk=16, n=1, dtype=BF16):
    return torch.zeros(b, n, h, dk, dtype=dtype)


def test_an_empty_ring():
    ring = _ring(3, 2, 24, 7)
    assert ring.k.shape == (3, 2, 7, 12) and ring.k_scale.shape == (3, 2, 7, 2) and ring.pos.shape == (3, 7)
    assert not any(bool(t.any()) for t in ring.tensors())


@pytest.mark.parametrize(("kwargs", "error", "match"), [
    ({"w": 0}, ValueError, "window"),
    ({"dk": 12}, ValueError, "head dimension 12"),
    ({"dk": 264}, ValueError, "head dimension 264"),
    ({"dk": 0}, ValueError, "head dimension 0"),
    ({"dtype": torch.float32}, ValueError, "dtype"),
])
def test_rings_outside_the_contract(kwargs, error, match):
    with pytest.raises(error, match=match):
        _ring(**kwargs)


def test_the_write_refuses():
    from vesper.contracts import ContractError
    from vesper.kernels.ring_quant import quant_ring_write

    k, pos, ring = _token(n=3), torch.arange(3).expand(2, 3), _ring()
    for bad, match in (((k[:, :2], k, pos, ring), "axis 1"), ((k, k.half(), pos, ring), "dtype"),
                       ((k, k, pos.int(), ring), "dtype"), ((k, k, pos, _ring(hkv=1)), "hkv"),
                       ((k, k, pos, _ring(dk=24)), "features"), ((k, k, pos, _ring(dtype=torch.float16)), "dtype"),
                       ((k, k, pos, _ring(b=3)), "'b'"), ((k, k, pos, ring), "CUDA only")):
        with pytest.raises(ContractError, match=match):
            quant_ring_write(*bad)


def test_the_read_refuses():
    from vesper.contracts import ContractError
    from vesper.kernels.ring_quant import QuantRingKVCache, quant_ring_read

    ring = _ring()
    with pytest.raises(ContractError, match="dtype"):
        quant_ring_read(ring, torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises(ContractError, match="'b'"):
        quant_ring_read(ring, torch.zeros(3, 3, dtype=torch.long))
    with pytest.raises(ContractError, match="CUDA only"):
        quant_ring_read(ring, torch.zeros(2, 3, dtype=torch.long))
    with pytest.raises(ContractError, match="'w'"):
        quant_ring_read(QuantRingKVCache(*ring.tensors(), 9), torch.zeros(2, 3, dtype=torch.long))
    with pytest.raises(ContractError, match="dtype"):
        quant_ring_read(QuantRingKVCache(ring.k.char(), *ring.tensors()[1:], 8), torch.zeros(2, 3, dtype=torch.long))


def test_the_attention_refuses():
    from vesper.contracts import ContractError
    from vesper.kernels.ring_quant import quant_ring_attention

    q, k, pos, ring = _token(h=4), _token(), torch.zeros(2, 1, dtype=torch.long), _ring()
    for bad, match in (((_token(n=2), k, k, pos, ring), "axis 1"), ((q.half(), k, k, pos, ring), "dtype"),
                       ((q, k, k, pos, _ring(dtype=torch.float16)), "dtype"), ((q, k, k, pos.int(), ring), "dtype"),
                       ((q, k, k, pos, ring), "CUDA only")):
        with pytest.raises(ContractError, match=match):
            quant_ring_attention(*bad)


def test_the_norm_and_the_projection_refuse():
    from vesper.contracts import ContractError
    from vesper.kernels.norm import projection_int8, quantize_weights, rms_norm_int8

    with pytest.raises(ContractError, match="CUDA only"):
        rms_norm_int8(torch.zeros(2, 64))
    z, w = torch.zeros(2, 64, dtype=torch.int8), torch.zeros(1, 8, 64, dtype=torch.int8)
    with pytest.raises(ContractError, match="CUDA"):
        projection_int8(z, torch.ones(2), w, torch.ones(1, 8), (8,))
    with pytest.raises(ContractError, match="floating"):
        quantize_weights(torch.zeros(2, 8, dtype=torch.float32))
    with pytest.raises(ContractError, match="floating"):
        quantize_weights(w)
    with pytest.raises(ContractError, match="finite"):
        quantize_weights(torch.full((1, 2, 16), math.nan))


def test_the_column_refuses_other_forms():
    from vesper.contracts import ContractError
    from vesper.decode import cold_states, per_pass
    from vesper.loop import LoopedColumn

    with pytest.raises(ValueError, match="projections"):
        LoopedColumn.random(32, 2, 1, 16, 4, 1, 0, torch.device("cpu"), projections="int4")
    with pytest.raises(ValueError, match="multiple of 16"):
        LoopedColumn.random(24, 3, 3, 8, 4, 1, 0, torch.device("cpu"), projections="int8")
    assert per_pass() == 6 and per_pass(4) == 8
    column = LoopedColumn.random(32, 2, 1, 16, 4, 2, 0, torch.device("cpu"), projections="int8")
    with pytest.raises(ContractError, match="ring_bits"):
        cold_states(column, 1, torch.device("cpu"), 8)
    flat = cold_states(column, 3, torch.device("cpu"), 4)
    assert len(flat) == 16 and flat[2].shape == (3, 1, 4, 8) and flat[4].shape == (3, 1, 4, 2)
    (codes, scale), _ = column.int8_weights(1)
    assert codes.shape == (4, 32, 32) and scale.shape == (4, 32)


def test_the_c_entries_refuse_before_any_launch():
    from vesper.kernels import _lib

    lib = _lib.library()
    none8, err = [None] * 10, lambda: lib.vsp_last_error().decode()  # noqa: E731
    one = 0x1000  # never read: the call is refused first
    write, read, attn = lib.vsp_quant_ring_write_bf16, lib.vsp_quant_ring_read_bf16, lib.vsp_quant_ring_attn_bf16
    assert write(*none8, 1, 1, 1, 12, 4, None) != 0 and "head dimension 12" in err()
    assert write(*none8, 1, -1, 1, 16, 4, None) != 0 and "N=-1" in err()
    assert write(*none8, 1, 1, 1, 16, 0, None) != 0 and "W=0" in err()
    assert write(*none8, 1, 1, 1, 16, 4, None) != 0 and "null" in err()
    assert write(*none8, 1, 1, 1, 256, 1 << 24, None) != 0 and "2 GiB" in err()
    assert write(one + 8, *[one] * 9, 1, 1, 1, 16, 4, None) != 0 and "16-byte" in err()
    assert write(one, one, one, None, one + 2, *[one] * 5, 1, 1, 1, 16, 4, None) != 0 and "4-byte" in err()
    assert write(*none8, 0, 1, 1, 16, 4, None) == 0 and write(*none8, 1, 0, 1, 16, 4, None) == 0
    assert write(*[one] * 10, 1 << 24, 1, 1, 16, 4, None) != 0 and "16777216 workgroups" in err()
    assert read(*[one] * 10, 1 << 24, 1, 1, 16, 4, None) != 0 and "16777216 workgroups" in err()
    assert read(*none8, 1, 1, 0, 16, 4, None) != 0 and "HKV=0" in err()
    assert read(*none8, 1, 1, 1, 16, 4, None) != 0 and "null" in err()
    assert read(*none8, 1, 0, 1, 16, 4, None) == 0
    call = lambda ptrs, b, h, hkv, d, w, ws=0: attn(*ptrs, ws, b, h, hkv, d, w, 1.0, 1, None)  # noqa: E731
    assert call([None] * 13, 1, 3, 2, 16, 4) != 0 and "multiple of 2" in err()
    assert call([None] * 13, 1, 9, 1, 16, 4) != 0 and "at most 8" in err()
    assert call([None] * 13, 1, 1, 1, 264, 4) != 0 and "264" in err()
    assert call([None] * 13, 1, 1, 1, 16, 4) != 0 and "null" in err()
    assert call([None] * 13, 0, 1, 1, 16, 4) == 0
    assert call([one] * 13, 1 << 24, 1, 1, 16, 4) != 0 and "workgroups" in err()
    need = lib.vsp_quant_ring_attn_workspace_bytes(1, 2, 1, 64, 4096)
    assert need > 0
    assert call([one] * 13, 1, 2, 1, 64, 4096, need - 1) != 0 and "workspace" in err()
    assert lib.vsp_quant_ring_attn_workspace_bytes(0, 2, 1, 64, 4096) == 0
    norm = lib.vsp_rms_norm_int8_f32_bf16
    assert norm(None, None, None, None, None, None, 1, 12, None) != 0 and "width 12" in err()
    assert norm(None, None, None, None, None, None, 1, 16392, None) != 0 and "16392" in err()
    assert norm(None, None, None, None, None, None, 1, 16, None) != 0 and "null" in err()
    assert norm(one, None, one, None, one, one, 1, 16, None) != 0 and "residual" in err()
    assert norm(one + 4, None, None, None, one, one, 1, 16, None) != 0 and "16-byte" in err()
    assert norm(None, None, None, None, None, None, 0, 16, None) == 0
    project = lib.vsp_project_int8_bf16
    args = lambda p=1, cols=8, d=64, m=4, used=(8, 1, 1, 1), outs=(None,) * 4, sig=-1: project(  # noqa: E731
        None, None, None, None, p, cols, d, m, *used, *outs, sig, None)
    assert args(p=5) != 0 and "weight blocks" in err()
    assert args(d=24) != 0 and "width 24" in err()
    assert args(d=16400) != 0 and "16400" in err()
    assert args(m=-1) != 0 and "M=-1" in err()
    assert args(sig=1) != 0 and "sigmoid" in err()
    assert args(used=(9, 1, 1, 1)) != 0 and "9 of its 8" in err()
    assert args() != 0 and "null output" in err()
    assert args(outs=(one + 8, None, None, None)) != 0 and "16-byte" in err()
    assert args(outs=(one, None, None, None)) != 0 and "null pointer" in err()
    assert args(m=0) == 0


def test_the_oracles_quantiser_on_a_row_done_by_hand():
    """[-1, 0.5, 2, 14]: scale 15 / 15 = 1, codes 0, 2 (1.5 to even), 3, 15."""
    from oracle.quant import quantize_rows, ring_values, row_values, unpack_rows

    x = torch.tensor([[-1.0, 0.5, 2.0, 14.0]], dtype=BF16)
    codes, scale, lo, t = quantize_rows(x)
    assert codes.tolist() == [[0, 2, 3, 15]] and scale.item() == 1 and lo.item() == -1 and t.tolist() == [[0, 1.5, 3, 15]]
    assert row_values(codes, scale, lo).tolist() == [[-1, 1, 2, 14]]
    packed = torch.tensor([[0x20, 0xF3]], dtype=torch.uint8)
    assert torch.equal(unpack_rows(packed), codes)
    assert ring_values(packed, torch.tensor([[1.0, -1.0]])).tolist() == [[-1, 1, 2, 14]]


TOO_MANY = 2**32 + 8  # cut to 32 bits these are 8: sizes that every other check would take


def _huge_ring(b, w, device="cpu"):
    """A ring of ``b`` rows and ``w`` slots of one head of eight features, broadcast: nothing of that size is allocated."""
    from vesper.kernels.ring_quant import QuantRingKVCache

    one = lambda *shape, dtype: torch.zeros(1, dtype=dtype, device=device).expand(*shape)  # noqa: E731
    return QuantRingKVCache(one(b, 1, w, 4, dtype=torch.uint8), one(b, 1, w, 4, dtype=torch.uint8), one(b, 1, w, 2, dtype=BF16),
                            one(b, 1, w, 2, dtype=BF16), one(b, w, dtype=torch.long), one(b, w, dtype=torch.bool), w)


@pytest.mark.parametrize(("b", "n", "w"), [(1, TOO_MANY, 4), (TOO_MANY, 1, 4), (1, 3, TOO_MANY), (2**31, 1, 4), (1, 2**31, 4)])
def test_ring_sizes_past_32_bits_are_refused(b, n, w):
    """The kernels count rows, tokens and slots in 32 bits: a size past them is refused, never cut."""
    from vesper.contracts import ContractError
    from vesper.kernels.ring_quant import quant_ring_attention, quant_ring_read, quant_ring_write

    tokens, pos = torch.zeros(1, dtype=BF16).expand(b, n, 1, 8), torch.zeros(1, dtype=torch.long).expand(b, n)
    ring = _huge_ring(b, w)
    with pytest.raises(ContractError, match="at most 2147483647"):
        quant_ring_write(tokens, tokens, pos, ring)
    with pytest.raises(ContractError, match="at most 2147483647"):
        quant_ring_read(ring, pos)
    if n != 1 and w == 4:
        return  # a step has one token a row
    token = tokens[:, :1]
    with pytest.raises(ContractError, match="at most 2147483647"):
        quant_ring_attention(token, token, token, pos[:, :1], ring)


def test_an_empty_ring_of_too_many_slots_is_refused():
    from vesper.contracts import ContractError
    from vesper.kernels.ring_quant import quant_ring_empty

    for b, w in ((1, TOO_MANY), (TOO_MANY, 4)):
        with pytest.raises(ContractError, match="at most 2147483647"):
            quant_ring_empty(b, 1, 8, w, BF16, torch.device("meta"))


def test_weights_of_too_many_columns_are_refused():
    """A column count cut to 32 bits would put every block after the first in the wrong place."""
    from vesper.contracts import ContractError
    from vesper.kernels.norm import projection_int8

    z, one = torch.zeros(2, 16, dtype=torch.int8), torch.ones(1)
    w = torch.zeros(1, dtype=torch.int8).expand(2, TOO_MANY, 16)
    with pytest.raises(ContractError, match="4294967304 columns, the kernel takes at most 2147483647"):
        projection_int8(z, one.expand(2), w, one.expand(2, TOO_MANY), (8, 8))


def test_a_few_token_launch_of_2_to_the_32_threads_is_refused():
    """2^28 columns in workgroups of 16 columns and 256 threads (one token), or of 32 and 512 (20 tokens): 2^32 threads."""
    from vesper.kernels import _lib

    lib, one = _lib.library(), 0x1000  # never read: the call is refused first
    for m, groups in ((1, 1 << 24), (20, 1 << 23)):
        status = lib.vsp_project_int8_bf16(one, one, one, one, 1, 1 << 28, 16, m, 1 << 28, 1, 1, 1, one, None, None, None, -1, None)
        assert status == 2 and f"{groups} workgroups" in lib.vsp_last_error().decode()


@pytest.mark.parametrize(("a", "b", "same"), [
    ((0, 64), (0, 64), True), ((0, 64), (8, 72), True), ((8, 72), (0, 64), True), ((0, 64), (63, 64), True),
    ((0, 64), (64, 128), False), ((64, 128), (0, 64), False), ((32, 32), (0, 64), False), ((0, 64), (32, 32), False),
])
def test_tensors_that_share_memory_in_part(a, b, same):
    from vesper.kernels.norm import _overlap

    buf = torch.zeros(128)
    assert _overlap(buf[slice(*a)], buf[slice(*b)]) is same
    assert _overlap(buf[slice(*a)], buf.view(BF16)[2 * b[0]:2 * b[1]]) is same


class _Placed:
    """A tensor as the norms' argument checks see one on a GPU (one that no machine has, so that no kernel is reached)."""

    def __init__(self, t):
        self.t = t

    device = torch.device("cuda", 99)

    def get_device(self):
        return 99

    def contiguous(self):
        return self

    def __getattr__(self, name):
        return getattr(self.t, name)


def test_a_sum_that_overlaps_an_input_in_part_is_refused():
    """One row's sum would overwrite what another row has yet to read."""
    from vesper.contracts import ContractError
    from vesper.kernels.norm import rms_norm_int8

    n, d = 4, 64
    buf, other = torch.zeros((n + 1) * d), torch.zeros(n, d, dtype=BF16)
    x, late, gain = _Placed(buf[:n * d].view(n, d)), _Placed(buf[d:].view(n, d)), _Placed(buf[n * d:])
    inside = _Placed(buf.view(BF16)[d:(n + 1) * d].view(n, d))
    apart = _Placed(torch.zeros(n, d))
    for kwargs in (dict(x=x, residual=_Placed(other), sum_out=late), dict(x=late, residual=_Placed(other), sum_out=x),
                   dict(x=apart, residual=inside, sum_out=x), dict(x=apart, residual=_Placed(other), gain=gain, sum_out=late)):
        with pytest.raises(ContractError, match="overlap"):
            rms_norm_int8(**kwargs)
