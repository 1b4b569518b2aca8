"""What the bf16 norm and the decode projection refuse of their sums' memory, on the CPU."""

from __future__ import annotations

import pytest
import torch

BF16 = torch.bfloat16


class _Placed:
    """A tensor as the argument checks see one on a GPU (one that no machine has, so that no kernel is reached)."""

    device = torch.device("cuda", 99)

    def __init__(self, t):
        self.t = t

    def contiguous(self):
        return self

    def __getattr__(self, name):
        return getattr(self.t, name)


@pytest.mark.parametrize("projects", [False, True])
def test_a_sum_that_overlaps_an_input_in_part_is_refused(projects):
    """One row's sum would overwrite what another row has yet to read."""
    from vesper.contracts import ContractError
    from vesper.kernels.norm import decode_projection, rms_norm_bf16

    n, d = 4, 64
    buf = torch.zeros((n + 1) * d)
    x, late, gain = _Placed(buf[:n * d].view(n, d)), _Placed(buf[d:].view(n, d)), _Placed(buf[n * d:])
    inside, apart = _Placed(buf.view(BF16)[d:(n + 1) * d].view(n, d)), _Placed(torch.zeros(n, d))
    other, w = _Placed(torch.zeros(n, d, dtype=BF16)), _Placed(torch.zeros(1, 8, d, dtype=BF16))
    call = (lambda x, **kw: decode_projection(x, kw.pop("w", w), (4,), **kw)) if projects else rms_norm_bf16
    cases = [dict(x=x, residual=other, sum_out=late), dict(x=late, residual=other, sum_out=x),
             dict(x=apart, residual=inside, sum_out=x), dict(x=apart, residual=other, gain=gain, sum_out=late)]
    if projects:
        cases.append(dict(x=apart, residual=other, sum_out=x, w=_Placed(buf.view(BF16)[:8 * d].view(1, 8, d))))
    for kwargs in cases:
        with pytest.raises(ContractError, match="overlap"):
            call(**kwargs)
