"""What the gated scan, its step and the layer norm refuse, on the CPU, before any kernel is reached; the column's
gated sublayer in its plain form."""

from __future__ import annotations

import math

import pytest
import torch

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class _Placed(torch.Tensor):
    """A CPU tensor that says it lies on a GPU (one that no machine has, so that no kernel is reached)."""

    @property
    def device(self):
        return torch.device("cuda", 99)


def _on(t):
    return t.as_subclass(_Placed)


def _args(lead=(2, 3), h=4, dk=8, dtype=BF16):
    q, k, v = (_on(torch.zeros(*lead, h, dk, dtype=dtype)) for _ in range(3))
    beta, g = _on(torch.zeros(*lead, h, dtype=dtype)), _on(torch.zeros(*lead, h))
    return dict(q=q, k=k, v=v, beta=beta, g=g, state=_on(torch.zeros(lead[0], h, dk, dk)))


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize(("name", "change", "match"), [
    ("q", lambda t: t.to(F16), "dtype"),
    ("k", lambda t: t.to(F32), "dtype"),
    ("beta", lambda t: t.to(F32), "dtype"),
    ("g", lambda t: t.to(BF16), "g: dtype"),
    ("state", lambda t: t.to(BF16), "dtype"),
    ("k", lambda t: t[..., :4], "dk"),
    ("v", lambda t: t[:1], "'b'"),
    ("g", lambda t: t[..., :2], "'h'"),
    ("state", lambda t: t[:, :2], "'h'"),
    ("state", lambda t: t.as_subclass(torch.Tensor), "is on"),
    ("g", lambda t: t.as_subclass(torch.Tensor), "is on"),
    ("beta", lambda t: t[..., None], "rank"),
])
def test_arguments_outside_the_contract(step, name, change, match):
    from vesper.contracts import ContractError
    from vesper.kernels.gated_scan import gated_delta_scan, gated_delta_step

    args = _args(lead=(2,) if step else (2, 3))
    args[name] = change(args[name])
    with pytest.raises(ContractError, match=match):
        (gated_delta_step if step else gated_delta_scan)(**args)


def test_the_cpu_wide_heads_and_masks():
    from vesper.contracts import ContractError
    from vesper.kernels.gated_scan import gated_delta_scan, gated_delta_step

    with pytest.raises(ContractError, match="CUDA only"):
        gated_delta_scan(**{n: t.as_subclass(torch.Tensor) for n, t in _args().items()})
    with pytest.raises(ContractError, match="exceeds"):
        gated_delta_scan(**_args(dk=257))
    with pytest.raises(ContractError, match="head dimension 0"):
        gated_delta_step(**_args(lead=(2,), dk=0))
    with pytest.raises(ContractError, match="active"):
        gated_delta_scan(**_args(), active=_on(torch.ones(2, 4, dtype=torch.bool)))
    with pytest.raises(ContractError, match="dtype"):
        gated_delta_scan(**_args(), active=_on(torch.ones(2, 3)))
    with pytest.raises(ContractError, match="dtype"):  # checked for no tokens too
        gated_delta_scan(**_args(lead=(2, 0)), active=_on(torch.ones(2, 0)))


def test_no_tokens_return_what_came():
    from vesper.kernels.gated_scan import gated_delta_scan

    args = _args(lead=(2, 0))
    o, after = gated_delta_scan(**args)
    assert o is args["q"] and after is args["state"]


def test_the_step_s_states():
    from vesper.contracts import ContractError
    from vesper.kernels.gated_scan import gated_delta_step

    args = _args(lead=(2,))
    with pytest.raises(ContractError, match="contiguous"):
        gated_delta_step(**{**args, "state": args["state"].transpose(2, 3)})
    with pytest.raises(ContractError, match="out_state"):
        gated_delta_step(**args, out_state=_on(torch.zeros(2, 4, 8, 4)))
    with pytest.raises(ContractError, match="out_state"):
        gated_delta_step(**args, out_state=torch.zeros(2, 4, 8, 8))
    buf = torch.zeros(2 * 4 * 64 + 64)
    first, second = _on(buf[:512].view(2, 4, 8, 8)), _on(buf[64:].view(2, 4, 8, 8))
    with pytest.raises(ContractError, match="overlap"):
        gated_delta_step(**{**args, "state": first}, out_state=second)
    args["v"].requires_grad_()
    with pytest.raises(ContractError, match="forward only"):
        gated_delta_step(**args)


@pytest.mark.parametrize(("call", "match"), [
    (dict(x=torch.zeros(2, 8)), "CUDA only"),
    (dict(x=_on(torch.zeros(2, 8, dtype=torch.float64))), "dtype"),
    (dict(x=_on(torch.zeros(2, 0))), "last axis"),
    (dict(x=_on(torch.zeros(2, 16385))), "last axis"),
    (dict(x=_on(torch.zeros(()))), "last axis"),
    (dict(gain=_on(torch.zeros(4))), "gain"),
    (dict(gain=_on(torch.zeros(8, dtype=BF16))), "gain"),
    (dict(gain=torch.zeros(8)), "gain"),
    (dict(bias=_on(torch.zeros(1, 8))), "bias"),
    (dict(residual=_on(torch.zeros(2, 4))), "residual"),
    (dict(residual=torch.zeros(2, 8)), "residual"),
    (dict(residual=_on(torch.zeros(2, 8, dtype=torch.float64))), "residual"),
    (dict(x=_on(torch.zeros(2, 8, dtype=BF16)), residual=_on(torch.zeros(2, 8))), "residual"),
    (dict(x=_on(torch.zeros(2, 8, dtype=BF16)), residual=_on(torch.zeros(2, 8, dtype=F16))), "residual"),
    (dict(x=_on(torch.zeros(2, 8, dtype=BF16)), dtype=F32), "dtype"),
    (dict(dtype=torch.float64), "dtype"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=math.nan), "eps"),
    (dict(eps=math.inf), "eps"),
])
def test_layer_norm_refusals(call, match):
    from vesper.contracts import ContractError
    from vesper.kernels.layer_norm import layer_norm

    with pytest.raises(ContractError, match=match):
        layer_norm(**{"x": _on(torch.zeros(2, 8)), "gain": _on(torch.zeros(8)), **call})


def test_the_c_entries_refuse_sizes_before_any_launch():
    from vesper.kernels import _lib

    lib = _lib.library()
    none = [None] * 9
    for sizes, text in (((1, 64, 1, 12), "head dimension"), ((1, 64, 1, 264), "head dimension"), ((1, 64, 1, 4), "head dimension"),
                        ((-1, 64, 1, 64), "bad sizes"), ((1, 64, 0, 64), "bad sizes"), ((0, 64, 1, 64), "no tokens"),
                        ((1, (1 << 30) + 1, 1, 64), "tokens a row"), ((1 << 20, 64 * 33, 1, 64), "chunks"),
                        ((1 << 20, 64, 1, 128), "slices"), ((1, 64, 1, 64), "null")):
        assert lib.vsp_gated_scan_bf16(*none, 0, None, 0, None, *sizes, None) != 0
        assert text in lib.vsp_last_error().decode(), sizes
    assert lib.vsp_gated_step_f32(*[None] * 9, 1 << 10, 1 << 10, 64, None) != 0 and "2^20" in lib.vsp_last_error().decode()
    assert lib.vsp_gated_step_f32(*[None] * 9, 1, 1, 300, None) != 0 and "head dimension" in lib.vsp_last_error().decode()
    assert lib.vsp_layer_norm(*[None] * 7, 1, 2, 1, 4, 8, 1e-5, None) != 0  # bfloat16 with a float16 residual
    assert lib.vsp_layer_norm(*[None] * 7, 0, 0, 0, 4, 16385, 1e-5, None) != 0 and "width" in lib.vsp_last_error().decode()
    # a workspace or records too small
    fake = [16] * 8
    assert lib.vsp_gated_scan_f32(*fake, 16, 64, None, 0, None, 1, 64, 1, 64, None) != 0 and "workspace" in lib.vsp_last_error().decode()
    need = lib.vsp_gated_scan_workspace_bytes(1, 64, 1, 64, 1)
    assert lib.vsp_gated_scan_f32(*fake, 16, need, 16, 64, None, 1, 64, 1, 64, None) != 0 and "records" in lib.vsp_last_error().decode()
    assert lib.vsp_gated_scan_f32(8, *fake[1:], 16, need, None, 0, None, 1, 64, 1, 64, None) != 0 and "aligned" in lib.vsp_last_error().decode()


def test_workspace_sizes():
    from vesper.kernels import _lib

    lib = _lib.library()
    assert lib.vsp_gated_scan_records_bytes(2, 130, 3, 64) == 2 * 3 * 3 * 64 * (64 + 64) * 4
    assert lib.vsp_gated_scan_records_bytes(0, 130, 3, 64) == 0
    assert lib.vsp_layer_norm_backward_workspace_bytes(10, 768) == 3 * 2 * 768 * 4
    assert lib.vsp_layer_norm_backward_workspace_bytes(0, 768) == 0


def test_a_sublayer_s_first_parameters_are_drawn_as_without_decay():
    from vesper.column import RecurrentSublayer

    plain = RecurrentSublayer(32, 4, key_conv=3, generator=torch.Generator().manual_seed(1))
    gated = RecurrentSublayer(32, 4, key_conv=3, generator=torch.Generator().manual_seed(1), decay=True, norm=True)
    shared = dict(gated.named_parameters())
    for name, p in plain.named_parameters():
        assert torch.equal(p, shared.pop(name)), name
    assert set(shared) == {"w_decay", "decay_rate", "norm_gain", "norm_bias"}
    x = torch.randn(2, 5, 32)
    assert plain.decays(x) is None and plain.normalize(x) is x
    g = gated.decays(x)
    assert g.shape == (2, 5, 4) and g.dtype == F32 and bool((g < 0).all())
    want = -torch.exp(gated.decay_rate) * torch.log1p(torch.exp(x @ gated.w_decay.t()))
    assert torch.allclose(g, want, rtol=1e-5, atol=1e-7)
    y = gated.normalize(x.to(BF16))
    assert y.dtype == BF16 and float(y.detach().float().mean(-1).abs().max()) < 2.0**-8 * 4


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_reference_scan_with_decays(dtype):
    from oracle.gated import gated_scan
    from vesper.column import recurrent_scan

    gen = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, 70, 3, 8, generator=gen).to(dtype) for _ in range(3))
    k = torch.nn.functional.normalize(k.float(), dim=-1).to(dtype)
    beta, g = torch.rand(2, 70, 3, generator=gen).to(dtype), -torch.rand(2, 70, 3, generator=gen)
    state = torch.randn(2, 3, 8, 8, generator=gen)
    o, after = recurrent_scan("reference", q, k, v, beta, state, g=g)
    want, last = gated_scan(*(t.double() for t in (q, k, v, beta, g, state)))
    assert o.dtype == dtype and after.dtype == F32
    assert float((o.double() - want).norm() / want.norm()) < (2.0**-8 if dtype == BF16 else 1e-5)
    assert float((after.double() - last).norm() / last.norm()) < 1e-5
