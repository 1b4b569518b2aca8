"""Layer norm on MI355X with the residual's addition in it, forward and backward (``vsp_layer_norm*``).

``layer_norm(x, gain, bias, residual=r)`` adds ``r`` to the residual stream ``x`` and normalizes the sum's rows for the
next sublayer, one launch; its backward pass gives the gradients of ``x``, ``r``, ``gain`` and ``bias`` in two (the
rows, then the sums over the rows).
"""

from __future__ import annotations

import functools
import math
from typing import Any

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from vesper.contracts import ContractError, refuse_tangents
from vesper.kernels import _lib

MAX_WIDTH = 16384
MAX_ROWS = 2**31 - 1  # the C entry counts rows in 32 bits
_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


@functools.lru_cache(maxsize=256)
def _workspace_bytes(rows: int, d: int) -> int:
    return int(_lib.library().vsp_layer_norm_backward_workspace_bytes(rows, d))


def _forward(x: Tensor, gain: Tensor, bias: Tensor | None, residual: Tensor | None, eps: float, dtype: torch.dtype,
             stats: Tensor | None) -> tuple[Tensor, Tensor]:
    """``(y, sum)`` of contiguous tensors; without a residual the sum is ``x`` itself."""
    d = x.shape[-1]
    y = torch.empty_like(x) if dtype is x.dtype else torch.empty_like(x, dtype=dtype)
    total = x if residual is None else torch.empty_like(x)
    code = _CODES[x.dtype]
    _lib.launch(x.device, "vsp_layer_norm", x.data_ptr(), None if residual is None else residual.data_ptr(), gain.data_ptr(),
                None if bias is None else bias.data_ptr(), None if residual is None else total.data_ptr(), y.data_ptr(),
                None if stats is None else stats.data_ptr(), code, code if residual is None else _CODES[residual.dtype],
                _CODES[dtype], x.numel() // d, d, eps)
    return y, total


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: Tensor, gain: Tensor, bias: Tensor | None, residual: Tensor | None, eps: float,
                dtype: torch.dtype) -> Any:  # noqa: D102
        ctx.set_materialize_grads(False)
        x, gain = x.contiguous(), gain.contiguous()
        bias = None if bias is None else bias.contiguous()
        residual = None if residual is None else residual.contiguous()
        stats = torch.empty((*x.shape[:-1], 2), dtype=torch.float32, device=x.device)
        y, total = _forward(x, gain, bias, residual, eps, dtype, stats)
        # a sum of 16 bits is formed again from x and the residual
        again = residual is not None and x.dtype != torch.float32
        ctx.save_for_backward(gain, stats, *((x, residual) if again else (total,)))
        ctx.residual = None if residual is None else residual.dtype
        ctx.dtype = dtype
        return y if residual is None else (y, total)

    @staticmethod
    def backward(ctx: Any, dy: Tensor | None, dsum: Tensor | None = None) -> tuple[Tensor | None, ...]:  # noqa: D102
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, dy, dsum)


def _backward(ctx: Any, dy: Tensor | None, dsum: Tensor | None) -> tuple[Tensor | None, ...]:
    gain, stats, total, *rest = ctx.saved_tensors
    d = gain.shape[0]
    rows = total.numel() // d
    dy = torch.zeros(total.shape, dtype=ctx.dtype, device=total.device) if dy is None else dy.contiguous()
    dsum = None if dsum is None else dsum.contiguous()
    dx, dgain, dbias = torch.empty_like(total), torch.empty_like(gain), torch.empty_like(gain)
    other = ctx.residual is not None and ctx.residual != total.dtype
    dres = torch.empty(total.shape, dtype=ctx.residual, device=total.device) if other else None
    ws_bytes = _workspace_bytes(rows, d)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=total.device)
    with _lib.on_device(total.device):
        _lib.call("vsp_layer_norm_backward", total.data_ptr(), _lib.ptr(rest[0] if rest else None), gain.data_ptr(),
                  stats.data_ptr(), dy.data_ptr(), _lib.ptr(dsum), dx.data_ptr(), _lib.ptr(dres), dgain.data_ptr(), dbias.data_ptr(), ws.data_ptr(),
                  ws_bytes, _CODES[total.dtype], _CODES[ctx.residual or total.dtype], _CODES[ctx.dtype], rows, d,
                  _lib.stream_of(total.device))
    need = ctx.needs_input_grad
    return (dx if need[0] else None, dgain if need[1] else None, dbias if need[2] else None,
            (dres if other else dx) if need[3] else None, None, None)


_backward_once = once_differentiable(_backward)  # under create_graph: its results refuse a derivative


def layer_norm(x: Tensor, gain: Tensor, bias: Tensor | None = None, *, residual: Tensor | None = None,
               eps: float = 1e-5, dtype: torch.dtype | None = None) -> Tensor | tuple[Tensor, Tensor]:
    """Layer norm over the last axis of ``x [..., d]``, or of the float32 sum ``s = x + residual``:
    ``(s - mean) / sqrt(var + eps) * gain + bias``, in float32, rounded once.

    Args:
        x: float32, bfloat16 or float16 on the GPU, ``d`` in 1..16384 (widths that are multiples of 8 are the fast ones).
        gain: float32 ``[d]``.
        bias: optional float32 ``[d]``.
        residual: optional tensor shaped like ``x``: of x's dtype, or with a float32 ``x`` of any of the three.
        eps: added to the variance; finite, not negative. With 0 a row without deviations is NaN (0 / 0), and gradients are
            finite from deviations of ``2 ** -120`` on.
        dtype: the norm's dtype, with a float32 ``x`` any of the three (by default x's).

    Returns:
        the norm ``y [..., d]``; with a residual ``(y, s)``, the sum rounded to x's dtype.

    Under autograd the gradients of ``x``, ``residual``, ``gain`` and ``bias`` (each in its input's dtype) come from the
    backward kernels, from the float32 sum; they may be captured into a graph, as long as no eager graph of the same leaves
    is alive (torch's accumulation into them would leave the capture). Rows of sums ``s`` below ``2 ** 126`` give finite
    norms, however large their own sum is.

    Raises:
        ContractError: on a dtype, width, shape or device outside that contract or a forward-mode tangent, before any kernel
            runs.
    """
    out = x.dtype if dtype is None else dtype
    d = _check(x, gain, bias, residual, eps, out)
    if forward_ad._current_level >= 0:  # noqa: SLF001
        refuse_tangents(x, gain, bias, residual)
    grad = torch.is_grad_enabled() and (x.requires_grad or gain.requires_grad or (bias is not None and bias.requires_grad)
                                        or (residual is not None and residual.requires_grad))
    if x.numel() == 0 or not grad:
        if x.numel() == 0:  # no rows: empty results that keep the graph
            total = x if residual is None else x + residual.to(x.dtype)
            y = (total * gain if bias is None else total * gain + bias).to(out)
            return y if residual is None else (y, total)
        y, total = _forward(x.contiguous(), gain.contiguous(), None if bias is None else bias.contiguous(),
                            None if residual is None else residual.contiguous(), eps, out, None)
        return y if residual is None else (y, total)
    return _LayerNorm.apply(x, gain, bias, residual, eps, out)


def _check(x: Tensor, gain: Tensor, bias: Tensor | None, residual: Tensor | None, eps: float, out: torch.dtype) -> int:
    """Raises for what ``layer_norm`` does not take; returns the width."""
    if x.dtype not in _CODES:
        raise ContractError(f"x: dtype must be float32, bfloat16 or float16, got {x.dtype}")
    if x.device.type != "cuda":
        raise ContractError(f"the norm kernel runs on CUDA only, x is on {x.device}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ContractError(f"x: needs a last axis in 1..{MAX_WIDTH}, got {tuple(x.shape)}")
    d = x.shape[-1]
    if x.numel() > MAX_ROWS * d:
        raise ContractError(f"x: {x.numel() // d} rows, the kernel takes at most {MAX_ROWS}")
    for name, t in (("gain", gain), ("bias", bias)):
        if t is not None and (t.shape != (d,) or t.dtype != torch.float32 or t.device != x.device):
            raise ContractError(f"{name}: must be float32 [{d}] on {x.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if residual is not None:
        if residual.shape != x.shape or residual.device != x.device:
            raise ContractError(f"residual: {tuple(x.shape)} on {x.device}, got {tuple(residual.shape)} on {residual.device}")
        if residual.dtype != x.dtype and (x.dtype != torch.float32 or residual.dtype not in _CODES):
            raise ContractError(f"residual: dtype must be {x.dtype}{' or one of 16 bits' if x.dtype == torch.float32 else ''}, "
                                f"got {residual.dtype}")
    if out != x.dtype and (x.dtype != torch.float32 or out not in _CODES):
        raise ContractError(f"dtype must be {x.dtype}{' or one of 16 bits' if x.dtype == torch.float32 else ''}, got {out}")
    if not (math.isfinite(eps) and eps >= 0):
        raise ContractError(f"eps must be finite and not negative, got {eps}")
    return d
