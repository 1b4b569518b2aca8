"""The few-bit serving operators restated in float64 on the CPU, from their definitions.

Rows of four-bit codes: with ``lo`` and ``hi`` a row's smallest and largest feature, ``scale`` is ``(hi - lo) /
15`` rounded to the cache's dtype, a feature's code is ``round((x - lo) / scale)`` held to 0..15 (0 where the
scale is 0) and its value ``lo + scale * code``. A row with an infinity or a NaN is NaN throughout.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor


def quantize_rows(x: Tensor) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """``(codes, scale, lo, t)`` in float64 of rows ``x [..., dk]`` (bf16 or fp16); ``t`` the codes before rounding."""
    f = x.double()
    lo, hi = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    scale = ((hi - lo) / 15).to(x.dtype).double()
    t = torch.where(scale > 0, (f - lo) / scale, torch.zeros_like(f))
    fine = torch.isfinite(f).all(-1, keepdim=True)
    nan = torch.full_like(lo, math.nan)
    codes = torch.where(fine, torch.round(t).clamp(0, 15), torch.zeros_like(t))
    return codes, torch.where(fine, scale, nan), torch.where(fine, lo, nan), t


def row_values(codes: Tensor, scale: Tensor, lo: Tensor) -> Tensor:
    return lo + scale * codes


def unpack_rows(packed: Tensor) -> Tensor:
    """Codes ``[..., dk]`` (float64) of packed bytes ``[..., dk / 2]``, the even feature in the low half."""
    p = packed.long()
    return torch.stack([p % 16, p // 16], -1).flatten(-2).double()


def ring_values(packed: Tensor, pair: Tensor) -> Tensor:
    """The float64 values of a ring's rows ``[..., dk]``."""
    return row_values(unpack_rows(packed), pair[..., 0:1].double(), pair[..., 1:2].double())


def quant_ring_attend(q: Tensor, k: Tensor, v: Tensor, pos: Tensor, keys: Tensor, values: Tensor, ring_pos: Tensor,
                      valid: Tensor, window: int) -> Tensor:
    """The new token's attention: ``q [b, 1, h, dk]``, ``k, v [b, 1, hkv, dk]``, ``pos [b, 1]``, the ring's values
    ``keys, values [b, hkv, window, dk]``; slots that are valid, at a position in ``(p - window, p]`` and not
    slot ``p % window``, and the token itself."""
    b, _, h, dk = q.shape
    hkv = k.shape[2]
    out = torch.empty(b, 1, h, dk, dtype=torch.float64)
    slots = torch.arange(window)
    for i in range(b):
        p = int(pos[i, 0])
        use = valid[i] & (ring_pos[i] <= p) & (ring_pos[i] > p - window) & (slots != p % window)
        for head in range(h):
            kv = head // (h // hkv)
            rows = torch.cat([keys[i, kv, use].double(), k[i, :, kv].double()])
            vals = torch.cat([values[i, kv, use].double(), v[i, :, kv].double()])
            out[i, 0, head] = torch.softmax(rows @ q[i, 0, head].double() / math.sqrt(dk), 0) @ vals
    return out
