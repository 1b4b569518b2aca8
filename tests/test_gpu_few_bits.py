"""The column served in few bits on the GPU: 8-bit projections in the looped column and its decoder, four-bit
rings in the decoder.

The wiring is proved bitwise (one pass against the same public operators called one by one; the captured step
against the eager one; the ring's rows against the float64 quantiser of the bf16 decoder's rows), the whole
against the float64 oracle. Bound of the latter: the bf16 path's 3e-2, and for each of a pass's two sublayers
1e-2 more: rows and weights of 8-bit codes with a largest element of about 2.5 to 3.5 deviations are off by
3.5 / 127 / sqrt(12) = 0.8 % of a deviation each.
"""

from __future__ import annotations

import pytest
import torch

from conftest import needs_gpu
from oracle import loop as ol
from oracle.delta import relative_error
from oracle.quant import quantize_rows, unpack_rows

pytestmark = [pytest.mark.gpu, needs_gpu]

GPU = torch.device("cuda")
F64 = torch.float64


def _column(key_conv, projections, passes=3, d=64, h=4, hkv=2, dk=16, w=8, seed=1, copy_forward="fused"):
    from vesper.loop import LoopedColumn

    return LoopedColumn.random(d, h, hkv, dk, w, passes, seed, GPU, key_conv=key_conv, projections=projections,
                               copy_forward=copy_forward)


def _weights(column):
    ws = {name: [t.to("cpu", F64) for t in column.w[name]] for name in column.w}
    taps = None if column.taps is None else [t.to("cpu", F64) for t in column.taps]
    return ol.MixerWeights(**ws, heads=column.heads, kv_heads=column.kv_heads, head_dim=column.head_dim,
                           window=column.window, taps=taps, rotary_base=column.rotary_base)


def _inputs(b, n, d, seed):
    return torch.randn(b, n, d, generator=torch.Generator().manual_seed(seed)).to(GPU)


def _at(i, b):
    return torch.full((b, 1), i, dtype=torch.long, device=GPU)


@pytest.mark.parametrize("projections", ["bf16", "int8"])
@pytest.mark.parametrize("ring_bits", [16, 4])
@pytest.mark.parametrize("key_conv", [0, 4])
def test_the_captured_step_equals_the_eager_one_bitwise(projections, ring_bits, key_conv):
    from vesper.decode import CapturedDecoder, cold_states, decode_step

    column = _column(key_conv, projections)
    b, n, depth = 3, 14, 2
    x = _inputs(b, n, 64, seed=2)
    decoder = CapturedDecoder(column, depth, ring_bits=ring_bits)
    for generation in range(2):
        flat, eager = decoder.start(b), cold_states(column, b, GPU, ring_bits)
        for i in range(n):
            y, flat = decoder.step(x[:, i:i + 1], _at(i, b), flat)
            want, *eager = decode_step(column, depth, [x[:, i:i + 1], _at(i, b), *eager], ring_bits=ring_bits)
            torch.cuda.synchronize()
            assert torch.equal(y, want), (generation, i)
            for mine, theirs in zip(flat, eager):
                assert torch.equal(mine, theirs), (generation, i)
    assert decoder.captures == 1 and decoder.replays == 2 * n - 3


@pytest.mark.parametrize("key_conv", [0, 4])
def test_a_decode_pass_is_its_operators_one_by_one(key_conv):
    """Depth 1 in few bits: norm, product, delta step, norm, product, rotary, ring, called by hand."""
    from vesper.attention import rotary_qk
    from vesper.decode import cold_states, decode_step
    from vesper.kernels.delta_scan import delta_scan_step_fused, delta_scan_step_keys
    from vesper.kernels.norm import projection_int8, rms_norm_int8
    from vesper.kernels.ring_quant import QuantRingKVCache, quant_ring_attention
    from vesper.loop import _normalize

    column = _column(key_conv, "int8")
    b, d, h, hkv, dk = 2, 64, 4, 2, 16
    flat = cold_states(column, b, GPU, 4)
    mine = [t.clone() for t in flat]
    x = _inputs(b, 20, d, seed=3)
    for i in range(20):
        y, *flat = decode_step(column, 1, [x[:, i:i + 1], _at(i, b), *flat], ring_bits=4)
        state, history, *ring = mine[:8]
        rec, attn = column.int8_weights(0)
        xs = x[:, i]
        q, z, v, beta = projection_int8(*rms_norm_int8(xs), *rec, (d, d, d, h), sigmoid_block=3)
        q, v = q.view(b, h, dk), v.view(b, h, dk)
        if key_conv:
            o = delta_scan_step_keys(q, z, v, beta, history, column.taps[0], state)
        else:
            o, _ = delta_scan_step_fused(q, _normalize(z.view(b, 1, d), h)[:, 0], v, beta, state, out_state=state)
        x1 = torch.empty_like(xs)
        codes, scale = rms_norm_int8(xs, residual=o.reshape(b, d), sum_out=x1)
        aq, ak, av = projection_int8(codes, scale, *attn, (d, hkv * dk, hkv * dk))
        aq, ak = rotary_qk(aq.view(b, 1, h, dk), ak.view(b, 1, hkv, dk), _at(i, b), column.rotary_base)
        a, _ = quant_ring_attention(aq, ak, av.view(b, 1, hkv, dk), _at(i, b), QuantRingKVCache(*ring, column.window),
                                    inplace=True)
        assert torch.equal(y[:, 0], x1 + a.reshape(b, d))
        for got, want in zip(flat[:8], mine[:8]):
            assert torch.equal(got, want)


def test_the_first_pass_ring_holds_the_bf16_rings_rows_quantised():
    from vesper.decode import cold_states, decode_step

    column = _column(4, "bf16")
    b, n = 2, 21
    x = _inputs(b, n, 64, seed=4)
    wide, few = cold_states(column, b, GPU), cold_states(column, b, GPU, 4)
    for i in range(n):
        _, *wide = decode_step(column, 1, [x[:, i:i + 1], _at(i, b), *wide])
        _, *few = decode_step(column, 1, [x[:, i:i + 1], _at(i, b), *few], ring_bits=4)
    for which in (2, 3):
        codes, scale, lo, _ = quantize_rows(wide[which].cpu().transpose(1, 2))
        assert torch.equal(unpack_rows(few[which].cpu()), codes)
        assert torch.equal(few[which + 2].cpu().double(), torch.cat([scale, lo], -1))
    assert torch.equal(wide[4], few[6]) and torch.equal(wide[5], few[7])


def test_the_int8_decode_matches_the_oracle():
    from vesper.decode import cold_states, decode_step

    column = _column(4, "int8", d=128, dk=32)
    b, n, depth = 2, 20, 2
    x = _inputs(b, n, 128, seed=5)
    flat = cold_states(column, b, GPU)
    weights = _weights(column)
    step, states = ol.mixer_decode_step(weights, depth), ol.cold_decode_states(weights, b, F64)
    for i in range(n):
        y, *flat = decode_step(column, depth, [x[:, i:i + 1], _at(i, b), *flat])
        want, states = step(x[:, i:i + 1].cpu().double(), torch.full((b, 1), i, dtype=torch.long), states)
        assert relative_error(y, want) < 3e-2 + 2 * depth * 1e-2, i


def _loop_inputs(column, b, n, key_conv, seed):
    g = torch.Generator().manual_seed(seed)
    d, h, dk, passes = column.heads * column.head_dim, column.heads, column.head_dim, column.passes
    x0 = torch.randn(b, n, d, generator=g).to(GPU)
    exits = [(torch.rand(b, n, generator=g) < 0.3).to(GPU) for _ in range(passes)]
    states = [(0.02 * torch.randn(b, h, dk, dk, generator=g)).to(GPU) for _ in range(passes)]
    histories = [torch.randn(b, key_conv - 1, d, generator=g).to(GPU) for _ in range(passes)] if key_conv else None
    return x0, states, exits, histories


@pytest.mark.parametrize("key_conv", [0, 4])
def test_the_int8_loop_fuses_the_copy_forward_bitwise_and_matches_the_oracle(key_conv):
    column = _column(key_conv, "int8", passes=4, d=128, h=2, hkv=2, dk=64, w=64, seed=5)
    where = _column(key_conv, "int8", passes=4, d=128, h=2, hkv=2, dk=64, w=64, seed=5, copy_forward="where")
    x0, states, exits, histories = _loop_inputs(column, 2, 200, key_conv, seed=6)
    got, other = column.forward(x0, states, exits, histories), where.forward(x0, states, exits, histories)
    assert torch.equal(got.y, other.y) and torch.equal(got.n_iters, other.n_iters)
    for a, b in zip(got.states, other.states):
        assert torch.equal(a, b)
    if key_conv:
        return
    want = ol.loop_forward(x0.cpu().double(), ol.mixer_column_step(_weights(column)), [s.cpu().double() for s in states],
                           [e.cpu() for e in exits])
    assert torch.equal(got.n_iters.cpu(), want.n_iters)
    assert relative_error(got.y, want.y) < 3e-2 + 2 * 4 * 1e-2


def test_the_few_bit_forms_reach_their_kernels(monkeypatch):
    from vesper.decode import cold_states, decode_step
    from vesper.kernels import _lib

    seen: list[str] = []
    real = _lib.call
    monkeypatch.setattr(_lib, "call", lambda name, *args: (seen.append(name), real(name, *args))[1])
    column = _column(4, "int8")
    decode_step(column, 1, [_inputs(2, 1, 64, 1), _at(0, 2), *cold_states(column, 2, GPU, 4)], ring_bits=4)
    assert seen == ["vsp_rms_norm_int8_f32_bf16", "vsp_project_int8_bf16", "vsp_delta_step_keys_bf16",
                    "vsp_rms_norm_int8_f32_bf16", "vsp_project_int8_bf16", "vsp_rotary_qk_bf16", "vsp_quant_ring_attn_bf16",
                    "vsp_residual_rows_where"]
    seen.clear()
    column.forward(*_loop_inputs(column, 1, 40, 4, seed=7))
    assert seen.count("vsp_rms_norm_int8_f32_bf16") == 2 * 3 and seen.count("vsp_project_int8_bf16") == 2 * 3
    assert "vsp_rms_norm_bf16" not in seen and "vsp_project_bf16" not in seen


def test_a_decoder_of_one_form_refuses_the_others_states():
    from vesper.contracts import ContractError
    from vesper.decode import CapturedDecoder, cold_states

    column = _column(0, "bf16")
    decoder = CapturedDecoder(column, 2, ring_bits=4)
    with pytest.raises(ContractError, match="state tensors"):
        decoder.step(_inputs(1, 1, 64, 1), _at(0, 1), cold_states(column, 1, GPU))
    with pytest.raises(ContractError, match="ring_bits"):
        CapturedDecoder(column, 2, ring_bits=8)
