"""CPU oracle of the gated delta rule and of the layer norm (test infrastructure only; see ``oracle/__init__.py``).

Per head the state ``H [dk, dk]`` (key rows, value columns) and per token the log decay ``g``:

    H' = e^g H + k u^T,   u = beta (v - e^g H^T k),   o = H'^T q

one token after the other, in the inputs' dtype (the tests use float64). The reference has neither operator: both are
restated from their definitions, the rule as ``oracle.delta``'s with the state faded first.
"""

from __future__ import annotations

import torch
from torch import Tensor


def gated_step(q: Tensor, k: Tensor, v: Tensor, beta: Tensor, g: Tensor, state: Tensor) -> tuple[Tensor, Tensor]:
    """One token: ``q, k, v [b, h, dk]``, ``beta, g [b, h]``, ``state [b, h, dk, dk]``; ``(o, state')``."""
    faded = torch.exp(g)[..., None, None] * state
    u = beta[..., None] * (v - (faded * k[..., :, None]).sum(-2))
    after = faded + k[..., :, None] * u[..., None, :]
    return (after * q[..., :, None]).sum(-2), after


def gated_scan(q: Tensor, k: Tensor, v: Tensor, beta: Tensor, g: Tensor, state: Tensor,
               active: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """``n`` tokens in turn (``q, k, v [b, n, h, dk]``); inactive tokens' outputs are zero."""
    outs = []
    for t in range(q.shape[1]):
        o, state = gated_step(q[:, t], k[:, t], v[:, t], beta[:, t], g[:, t], state)
        outs.append(o)
    o = torch.stack(outs, 1) if outs else q
    return (o if active is None else o * active[:, :, None, None].to(o.dtype)), state


def layer_norm(x: Tensor, gain: Tensor, bias: Tensor | None, residual: Tensor | None, eps: float) -> tuple[Tensor, Tensor]:
    """``((s - mean) / sqrt(var + eps) gain + bias, s)`` of ``s = x + residual`` over the last axis."""
    s = x if residual is None else x + residual
    centred = s - s.mean(-1, keepdim=True)
    y = centred / torch.sqrt((centred * centred).mean(-1, keepdim=True) + eps) * gain
    return (y if bias is None else y + bias), s
