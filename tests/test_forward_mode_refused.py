"""Forward-mode derivatives: the scans, the step and the layer norm have none, and refuse inputs with a tangent, whether or not
one of them wants a gradient. On the CPU: no kernel is reached."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from test_gated_limits import _Wide, reached  # noqa: F401

BF16, F32 = torch.bfloat16, torch.float32


def _on(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Wide)


def _scan_args(dtype=F32, lead=(2, 3), h=2, dk=16):
    return [*(_on(*lead, h, dk, dtype=dtype) for _ in range(3)), _on(*lead, h, dtype=dtype), _on(*lead, h), _on(lead[0], h, dk, dk)]


def _dual(args, which):
    return [forward_ad.make_dual(t, torch.ones_like(t)) if i == which else t for i, t in enumerate(args)]


@pytest.mark.parametrize("lead", [(2, 3), (2, 1)])
@pytest.mark.parametrize("which", range(6))
def test_the_gated_scan(reached, lead, which):  # noqa: F811
    from vesper.contracts import ContractError
    from vesper.kernels.gated_scan import gated_delta_scan

    with forward_ad.dual_level():
        with pytest.raises(ContractError, match="forward-mode"):
            gated_delta_scan(*_dual(_scan_args(lead=lead), which))
        with torch.no_grad(), pytest.raises(ContractError, match="forward-mode"):
            gated_delta_scan(*_dual(_scan_args(lead=lead), which))
    assert not reached


@pytest.mark.parametrize("which", range(6))
def test_the_gated_step(reached, which):  # noqa: F811
    from vesper.contracts import ContractError
    from vesper.kernels.gated_scan import gated_delta_step

    args = [t[:, 0] for t in _scan_args()[:5]] + [_on(2, 2, 16, 16)]
    with forward_ad.dual_level(), pytest.raises(ContractError, match="forward-mode"):
        gated_delta_step(*_dual(args, which))
    assert not reached
    with forward_ad.dual_level():  # a level with no tangents
        gated_delta_step(*args)
    assert len(reached) == 1


@pytest.mark.parametrize("which", range(4))
def test_the_layer_norm(reached, which):  # noqa: F811
    from vesper.contracts import ContractError
    from vesper.kernels.layer_norm import layer_norm

    args = [_on(4, 16), _on(16), _on(16), _on(4, 16)]
    with forward_ad.dual_level(), pytest.raises(ContractError, match="forward-mode"):
        x, gain, bias, residual = _dual(args, which)
        layer_norm(x, gain, bias, residual=residual)
    assert not reached
    with forward_ad.dual_level():
        layer_norm(*args[:3], residual=args[3])
    assert len(reached) == 1


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("entry", ["delta_scan_fused", "delta_scan_fused_fp32", "delta_scan_step_fused"])
def test_the_delta_scans(entry, which):
    from vesper.contracts import ContractError
    from vesper.kernels import delta_scan

    args = _scan_args(BF16 if entry == "delta_scan_fused" else F32)
    args = args[:4] + args[5:]
    if "step" in entry:
        args = [t[:, 0] for t in args[:4]] + [_on(2, 2, 16, 16)]
    with forward_ad.dual_level(), pytest.raises(ContractError, match="forward-mode"):
        getattr(delta_scan, entry)(*_dual(args, which))


@pytest.mark.parametrize("which", range(3))
def test_the_delta_scan_s_carried_inputs(which):
    from vesper.contracts import ContractError
    from vesper.kernels.delta_scan import delta_scan_fused

    args = _scan_args(BF16)
    args = args[:4] + args[5:]
    with forward_ad.dual_level(), pytest.raises(ContractError, match="forward-mode"):
        delta_scan_fused(*args, active=_on(2, 3, dtype=torch.bool), carried=tuple(_dual([t.clone() for t in args[1:4]], which)))
