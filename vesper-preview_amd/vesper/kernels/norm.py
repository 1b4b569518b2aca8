"""The looped column's sublayer pre-normalization on MI355X: ``RMSNorm`` of float32 rows to bf16.

``rms_norm_bf16(x, gain)`` is ``RMSNorm.forward`` (``vesper/column.py:146-188``) on the float32
residual stream, ``x / sqrt(mean(x^2) + 1e-6) * gain`` computed scale-safely as the reference does,
returned in bfloat16 for the bf16 projection GEMMs (``vsp_rms_norm_bf16``, one launch).
``rms_norm_int8`` returns it in 8-bit integers with a scale a row (``vsp_rms_norm_int8_*``), the operand
of ``projection_int8`` (``vsp_project_int8_*``), whose weights ``quantize_weights`` lays out once.
"""

from __future__ import annotations

import torch
from torch import Tensor

from vesper.contracts import ContractError
from vesper.kernels import _lib


def rms_norm_bf16(x: Tensor, gain: Tensor | None = None, *, residual: Tensor | None = None,
                  sum_out: Tensor | None = None) -> Tensor:
    """``RMSNorm`` over the last axis of float32 ``x [..., d]`` on the GPU, as bfloat16.

    Args:
        x: float32, its last axis ``d`` a multiple of 8 in 8..2048.
        gain: optional float32 ``[d]`` (the norm's weight; ones when omitted).
        residual: optional bfloat16 tensor shaped like ``x``: the norm is then of ``x + residual``
            (added in float32, the column's residual add), in the same launch
            (``vsp_add_rms_norm_bf16``), bitwise the add followed by the norm.
        sum_out: with ``residual``, an optional contiguous float32 tensor shaped like ``x`` that receives
            ``x + residual``. It shares no memory with ``x``, ``residual`` or ``gain``.

    Raises:
        ContractError: on a dtype, width or device outside that contract.
    """
    if x.dtype != torch.float32:
        raise ContractError(f"x: dtype must be torch.float32, got {x.dtype}")
    if x.device.type != "cuda":
        raise ContractError(f"the norm kernel runs on CUDA only, x is on {x.device}")
    d = x.shape[-1]
    if d < 8 or d > 2048 or d % 8:
        raise ContractError(f"x: last axis {d} is not a multiple of 8 in 8..2048")
    xc = x.contiguous()
    if xc.data_ptr() % 16:
        xc = xc.clone()
    g = None
    if gain is not None:
        if gain.shape != (d,) or gain.dtype != torch.float32 or gain.device != x.device:
            raise ContractError(f"gain: must be float32 [{d}] on {x.device}, got {tuple(gain.shape)} {gain.dtype}")
        g = gain.contiguous()
        if g.data_ptr() % 16:
            g = g.clone()
    rows = xc.numel() // d
    if residual is None:
        if sum_out is not None:
            raise ContractError("sum_out needs a residual")
        out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
        with _lib.on_device(x.device):
            _lib.call("vsp_rms_norm_bf16", xc.data_ptr(), _lib.ptr(g), out.data_ptr(), rows, d,
                      _lib.stream_of(x.device))
        return out
    if residual.shape != x.shape or residual.dtype != torch.bfloat16 or residual.device != x.device:
        raise ContractError(f"residual: bf16 {tuple(x.shape)} on {x.device}, got {tuple(residual.shape)} "
                            f"{residual.dtype} on {residual.device}")
    rc = residual.contiguous()
    if rc.data_ptr() % 16:
        rc = rc.clone()
    if sum_out is not None:
        if (sum_out.shape != x.shape or sum_out.dtype != torch.float32 or sum_out.device != x.device
                or not sum_out.is_contiguous() or sum_out.data_ptr() % 16):
            raise ContractError(f"sum_out: contiguous, aligned float32 {tuple(x.shape)} on {x.device}")
        if _overlap(sum_out, xc) or _overlap(sum_out, rc) or (g is not None and _overlap(sum_out, g)):
            raise ContractError("sum_out must not be x, the residual or gain, nor overlap them")
    out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    with _lib.on_device(x.device):
        _lib.call("vsp_add_rms_norm_bf16", xc.data_ptr(), rc.data_ptr(), _lib.ptr(sum_out), _lib.ptr(g),
                  out.data_ptr(), rows, d, _lib.stream_of(x.device))
    return out


def decode_projection(x: Tensor, weights_t: Tensor, used: tuple[int, ...], *, residual: Tensor | None = None,
                      sum_out: Tensor | None = None, gain: Tensor | None = None,
                      sigmoid_block: int | None = None,
                      rotary: tuple[Tensor, Tensor, int, tuple[int, ...]] | None = None) -> list[Tensor]:
    """A decode step's sublayer projections in one launch (``vsp_decode_proj_bf16``): the residual
    sum ``s = x + residual`` (written into ``sum_out`` when given), ``z = RMSNorm(s, gain)`` in
    bfloat16 exactly as ``rms_norm_bf16`` computes it, and ``z W_j[:, :used_j]`` for each block of
    the stacked projection weight (``vesper/column.py:192-260``, ``vesper/attention.py:269-292``).

    Args:
        x: float32 ``[M, d]`` (one row a token), ``d`` a multiple of 32 in 32..2048.
        weights_t: bf16 ``[p, cols, d]``: the stacked ``[p, d, cols]`` weight, each block transposed.
        used: the columns kept of each of the ``p`` (1..4) blocks.
        residual: optional bf16 ``[M, d]`` added to ``x`` (the previous mixer's output).
        sum_out: optional float32 ``[M, d]`` that receives ``s``. It shares no memory with the other operands.
        gain: optional float32 ``[d]`` (the norm's weight; ones when omitted).
        sigmoid_block: the block whose outputs pass through the logistic function (the write strength).
        rotary: ``(positions, inv_freq, dk, blocks)``: the blocks rotated as they are stored, as
            ``rotary_qk`` rotates queries and keys (heads of ``dk`` columns, token ``m`` at
            ``positions[m]`` int64 ``[M]``, ``inv_freq`` the float64 ``[dk / 2]`` table), bitwise
            the separate launch's result.

    Returns:
        one bf16 ``[M, used_j]`` tensor per block.

    Raises:
        ContractError: on shapes, dtypes or devices outside that contract.
    """
    if x.dim() != 2 or x.dtype != torch.float32 or x.device.type != "cuda":
        raise ContractError(f"x: float32 [M, d] on CUDA, got {tuple(x.shape)} {x.dtype} on {x.device}")
    m, d = x.shape
    if weights_t.dim() != 3 or weights_t.dtype != torch.bfloat16 or weights_t.shape[2] != d:
        raise ContractError(f"weights_t: bf16 [p, cols, {d}], got {tuple(weights_t.shape)} {weights_t.dtype}")
    p, cols = weights_t.shape[0], weights_t.shape[1]
    if len(used) != p or not 1 <= p <= 4 or any(not 1 <= u <= cols for u in used):
        raise ContractError(f"used: {p} widths in 1..{cols}, got {tuple(used)}")
    if d % 32 or not 32 <= d <= 2048:
        raise ContractError(f"x: width {d} is not a multiple of 32 in 32..2048")
    tensors = [("weights_t", weights_t)]
    if residual is not None:
        if residual.shape != (m, d) or residual.dtype != torch.bfloat16:
            raise ContractError(f"residual: bf16 [{m}, {d}], got {tuple(residual.shape)} {residual.dtype}")
        tensors.append(("residual", residual))
    if sum_out is not None:
        if sum_out.shape != (m, d) or sum_out.dtype != torch.float32 or not sum_out.is_contiguous():
            raise ContractError(f"sum_out: contiguous float32 [{m}, {d}], got {tuple(sum_out.shape)} {sum_out.dtype}")
        tensors.append(("sum_out", sum_out))
    if gain is not None:
        if gain.shape != (d,) or gain.dtype != torch.float32:
            raise ContractError(f"gain: float32 [{d}], got {tuple(gain.shape)} {gain.dtype}")
        tensors.append(("gain", gain))
    for name, t in tensors:
        if t.device != x.device:
            raise ContractError(f"{name} is on {t.device}, x on {x.device}")
    if sigmoid_block is not None and not 0 <= sigmoid_block < p:
        raise ContractError(f"sigmoid_block {sigmoid_block} is not one of the {p} blocks")
    rot_pos, rot_freq, rot_dk, rot_mask = None, None, 0, 0
    if rotary is not None:
        rot_pos, rot_freq, rot_dk, blocks = rotary
        if rot_pos.shape != (m,) or rot_pos.dtype != torch.long or rot_pos.device != x.device:
            raise ContractError(f"rotary positions: int64 [{m}] on {x.device}, got {tuple(rot_pos.shape)} {rot_pos.dtype}")
        if rot_freq.shape != (rot_dk // 2,) or rot_freq.dtype != torch.float64 or rot_freq.device != x.device:
            raise ContractError(f"rotary frequencies: float64 [{rot_dk // 2}] on {x.device}")
        for j in blocks:
            if not 0 <= j < p or used[j] % rot_dk or j == sigmoid_block:
                raise ContractError(f"block {j} cannot be rotated in heads of {rot_dk}")
            rot_mask |= 1 << j
        rot_pos, rot_freq = rot_pos.contiguous(), rot_freq.contiguous()
    xc, wc = x.contiguous(), weights_t.contiguous()
    rc = None if residual is None else residual.contiguous()
    gc = None if gain is None else gain.contiguous()
    for name, t in (("x", xc), ("weights_t", wc), ("residual", rc), ("sum_out", sum_out), ("gain", gc)):
        if t is not None and t.data_ptr() % 16:
            raise ContractError(f"{name} must be 16-byte aligned")
    if sum_out is not None:
        for name, t in (("x", xc), ("residual", rc), ("gain", gc), ("weights_t", wc)):
            if t is not None and _overlap(sum_out, t):
                raise ContractError(f"sum_out must not be x or another operand, nor overlap one: it overlaps {name}")
    outs = [torch.empty(m, u, dtype=torch.bfloat16, device=x.device) for u in used]
    ptrs = [o.data_ptr() for o in outs] + [0] * (4 - p)
    widths = list(used) + [1] * (4 - p)
    with _lib.on_device(x.device):
        _lib.call("vsp_decode_proj_bf16", xc.data_ptr(), _lib.ptr(rc), _lib.ptr(sum_out), _lib.ptr(gc), wc.data_ptr(),
                  p, cols, d, m, *widths, *ptrs, -1 if sigmoid_block is None else sigmoid_block,
                  _lib.ptr(rot_pos), _lib.ptr(rot_freq), rot_mask, rot_dk, _lib.stream_of(x.device))
    return outs


def projection(z: Tensor, weights_t: Tensor, used: tuple[int, ...], *,
               sigmoid_block: int | None = None) -> list[Tensor]:
    """A prefill's sublayer projections in one launch (``vsp_project_bf16``): ``z W_j[:, :used_j]``
    for each block of the stacked projection weight (``vesper/column.py:192-260``,
    ``vesper/attention.py:269-292``), each block computed over the columns it uses only.

    Args:
        z: bf16 ``[M, d]``, the normalized input (one row a token), ``d`` a multiple of 64 in
            64..16384.
        weights_t: bf16 ``[p, cols, d]``: the stacked ``[p, d, cols]`` weight, each block transposed.
        used: the columns kept of each of the ``p`` (1..4) blocks.
        sigmoid_block: the block whose outputs pass through the logistic function (the write
            strength), as ``decode_projection`` stores it.

    Returns:
        one bf16 ``[M, used_j]`` tensor per block.

    Raises:
        ContractError: on shapes, dtypes or devices outside that contract.
    """
    if z.dim() != 2 or z.dtype != torch.bfloat16 or z.device.type != "cuda":
        raise ContractError(f"z: bf16 [M, d] on CUDA, got {tuple(z.shape)} {z.dtype} on {z.device}")
    m, d = z.shape
    if weights_t.dim() != 3 or weights_t.dtype != torch.bfloat16 or weights_t.shape[2] != d:
        raise ContractError(f"weights_t: bf16 [p, cols, {d}], got {tuple(weights_t.shape)} {weights_t.dtype}")
    if weights_t.device != z.device:
        raise ContractError(f"weights_t is on {weights_t.device}, z on {z.device}")
    p, cols = weights_t.shape[0], weights_t.shape[1]
    if len(used) != p or not 1 <= p <= 4 or any(not 1 <= u <= cols for u in used):
        raise ContractError(f"used: {p} widths in 1..{cols}, got {tuple(used)}")
    if d % 64 or not 64 <= d <= 16384:
        raise ContractError(f"z: width {d} is not a multiple of 64 in 64..16384")
    if (m + 256) * d * 2 >= 1 << 32 or (cols + 256) * d * 2 >= 1 << 32:
        raise ContractError(f"z [{m}, {d}] or a weight block of {cols} columns over 4 GiB")
    if sigmoid_block is not None and not 0 <= sigmoid_block < p:
        raise ContractError(f"sigmoid_block {sigmoid_block} is not one of the {p} blocks")
    zc, wc = z.contiguous(), weights_t.contiguous()
    for name, t in (("z", zc), ("weights_t", wc)):
        if t.data_ptr() % 16:
            raise ContractError(f"{name} must be 16-byte aligned")
    outs = [torch.empty(m, u, dtype=torch.bfloat16, device=z.device) for u in used]
    ptrs = [o.data_ptr() for o in outs] + [0] * (4 - p)
    widths = list(used) + [1] * (4 - p)
    with _lib.on_device(z.device):
        _lib.call("vsp_project_bf16", zc.data_ptr(), wc.data_ptr(), p, cols, d, m, *widths, *ptrs,
                  -1 if sigmoid_block is None else sigmoid_block, _lib.stream_of(z.device))
    return outs


MAX_ROWS = 2**31 - 1  # of the 8-bit operators: their C entries count rows and a weight's columns in 32 bits
_INT8_SUFFIX = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}
# x and residual dtypes of rms_norm_int8
_NORM_INT8 = {(torch.float32, torch.bfloat16): "f32_bf16", (torch.float32, torch.float16): "f32_f16",
              (torch.bfloat16, torch.bfloat16): "bf16", (torch.float16, torch.float16): "f16"}


def _aligned(t: Tensor, nbytes: int = 16) -> Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % nbytes == 0 else t.clone()


def _overlap(a: Tensor, b: Tensor) -> bool:
    """Whether two contiguous tensors share a byte."""
    s, t = a.data_ptr(), b.data_ptr()
    return s < t + b.nbytes and t < s + a.nbytes and a.numel() > 0 and b.numel() > 0


def _refuse_grad(name: str, *tensors: Tensor | None) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ContractError(f"{name} is forward only: call it under torch.no_grad()")


def rms_norm_int8(x: Tensor, gain: Tensor | None = None, *, residual: Tensor | None = None,
                  sum_out: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """``RMSNorm`` over the last axis of ``x [..., d]`` (plus ``residual``) in 8-bit integers, one scale a row:
    ``(codes int8 [..., d], scale float32 [...])`` with the norm ``y`` held as ``codes * scale``, ``scale = max
    |y| / 127`` and ``codes = round(y / scale)``, in one launch (``vsp_rms_norm_int8_*``). The arithmetic is float32: a
    quotient within 1e-3 of the middle between two codes may become either.

    Args:
        x: float32, bfloat16 or float16, its last axis ``d`` a multiple of 8 in 8..16384.
        gain: optional float32 ``[d]`` (the norm's weight; ones when omitted).
        residual: optional tensor shaped like ``x``, bfloat16 or float16 with a float32 ``x`` and else of x's
            dtype: the norm is of the float32 sum ``x + residual``.
        sum_out: with ``residual``, an optional contiguous tensor of x's shape and dtype that receives the sum,
            rounded to that dtype. It shares no memory with ``x``, ``residual`` or ``gain``: one row's sum is
            written while others are still read.

    A row whose normalized values are all below ``2 ** -120`` has scale 0 and codes 0; a row with an infinity
    or a NaN has scale NaN and codes 0.

    Raises:
        ContractError: on a dtype, width or device outside that contract, or a tensor that needs a gradient.
    """
    dtype, shape, device = x.dtype, x.shape, x.get_device()
    rdtype = (torch.bfloat16 if dtype is torch.float32 else dtype) if residual is None else residual.dtype
    suffix = _NORM_INT8.get((dtype, rdtype))
    d = shape[-1] if shape else 0
    # one test on the common path; the checks that name what is wrong run where it fails
    if not (suffix is not None and device >= 0 and 8 <= d <= 16384 and d & 7 == 0 and x.numel() <= MAX_ROWS * d
            and not x.requires_grad
            and (gain is None or (gain.shape == (d,) and gain.dtype is torch.float32 and gain.get_device() == device
                                  and not gain.requires_grad))
            and (residual is None or (residual.shape == shape and residual.get_device() == device
                                      and not residual.requires_grad))):
        _check_norm_int8(x, gain, residual, rdtype)
    xc = _aligned(x)
    gain = None if gain is None else _aligned(gain)
    residual = None if residual is None else _aligned(residual)
    if sum_out is not None:
        if residual is None:
            raise ContractError("sum_out needs a residual")
        if (sum_out.shape != shape or sum_out.dtype is not dtype or sum_out.get_device() != device
                or not sum_out.is_contiguous() or sum_out.data_ptr() % 16):
            raise ContractError(f"sum_out: contiguous, aligned {dtype} {tuple(shape)} on {x.device}")
        if _overlap(sum_out, xc) or _overlap(sum_out, residual) or (gain is not None and _overlap(sum_out, gain)):
            raise ContractError("sum_out must not be x, the residual or gain, nor overlap them")
    on = x.device
    codes = torch.empty(shape, dtype=torch.int8, device=on)
    scale = torch.empty(shape[:-1], dtype=torch.float32, device=on)
    with _lib.on_device(on):
        _lib.call(f"vsp_rms_norm_int8_{suffix}", xc.data_ptr(), _lib.ptr(residual), _lib.ptr(sum_out), _lib.ptr(gain),
                  codes.data_ptr(), scale.data_ptr(), xc.numel() // d, d, _lib.stream_of(on))
    return codes, scale


def _check_norm_int8(x: Tensor, gain: Tensor | None, residual: Tensor | None, rdtype: torch.dtype) -> None:
    """Raises for what ``rms_norm_int8`` does not take."""
    if x.device.type != "cuda":
        raise ContractError(f"the norm kernel runs on CUDA only, x is on {x.device}")
    if x.dim() < 1:
        raise ContractError("x: needs at least one axis")
    if (x.dtype, rdtype) not in _NORM_INT8:
        raise ContractError(f"x: dtype must be float32 (residual bfloat16 or float16), bfloat16 or float16 (residual the same), "
                            f"got {x.dtype} and {rdtype}")
    d = x.shape[-1]
    if d < 8 or d > 16384 or d % 8:
        raise ContractError(f"x: last axis {d} is not a multiple of 8 in 8..16384")
    if x.numel() > MAX_ROWS * d:
        raise ContractError(f"x: {x.numel() // d} rows, the kernel takes at most {MAX_ROWS}")
    _refuse_grad("rms_norm_int8", x, gain, residual)
    if gain is not None and (gain.shape != (d,) or gain.dtype != torch.float32 or gain.device != x.device):
        raise ContractError(f"gain: must be float32 [{d}] on {x.device}, got {tuple(gain.shape)} {gain.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.device != x.device):
        raise ContractError(f"residual: {tuple(x.shape)} on {x.device}, got {tuple(residual.shape)} on {residual.device}")


def quantize_weights(weights_t: Tensor) -> tuple[Tensor, Tensor]:
    """A stacked projection weight ``[p, cols, d]`` (each block transposed, one output channel a row) as the
    operands of ``projection_int8``, made once: int8 ``[p, cols, d]`` and float32 scales ``[p, cols]``, each row
    ``codes * scale`` with ``scale = max |w| / 127`` and ``codes = round(w / scale)`` (zeros for a row of zeros). Reads
    a flag back from the device, so it does not run under a graph capture.

    Raises:
        ContractError: if ``weights_t`` is not a floating ``[p, cols, d]`` tensor of finite values.
    """
    if weights_t.dim() != 3 or not weights_t.is_floating_point():
        raise ContractError(f"weights_t: floating [p, cols, d], got {tuple(weights_t.shape)} {weights_t.dtype}")
    with torch.no_grad():
        w = weights_t.float()
        if not bool(torch.isfinite(w).all()):
            raise ContractError("weights_t: every value must be finite")
        scale = w.abs().amax(-1) / 127 if w.shape[-1] else w.new_zeros(w.shape[:-1])
        codes = torch.where(scale[..., None] > 0, torch.round(w / scale[..., None]).clamp(-127, 127), torch.zeros_like(w))
        return codes.to(torch.int8).contiguous(), scale.contiguous()


def projection_int8(z: Tensor, z_scale: Tensor, weights_q: Tensor, weights_scale: Tensor, used: tuple[int, ...], *,
                    sigmoid_block: int | None = None, dtype: torch.dtype = torch.bfloat16) -> list[Tensor]:
    """A sublayer's projections in 8-bit integers (``vsp_project_int8_*``, one launch): for each block ``j`` of
    the stacked weight the sums of ``z[m, k] * weights_q[j, c, k]`` in int32 (exact) times ``z_scale[m] *
    weights_scale[j, c]``, over the columns it uses. The counterpart of ``projection`` and, with few tokens, of
    ``decode_projection``.

    Args:
        z: int8 ``[M, d]`` (``rms_norm_int8``'s codes, one row a token), ``d`` a multiple of 16 in 16..16384.
        z_scale: float32 ``[M]``.
        weights_q: int8 ``[p, cols, d]``: ``quantize_weights`` of the stacked ``[p, d, cols]`` weight, each block
            transposed.
        weights_scale: float32 ``[p, cols]``.
        used: the columns kept of each of the ``p`` (1..4) blocks.
        sigmoid_block: the block whose outputs pass through the logistic function (the write strength).
        dtype: the outputs' dtype: bfloat16, float16 or float32.

    Returns:
        one ``[M, used_j]`` tensor per block.

    Raises:
        ContractError: on shapes, dtypes or devices outside that contract, or a tensor that needs a gradient.
    """
    p = len(used)
    zshape, wshape, device, suffix = z.shape, weights_q.shape, z.get_device(), _INT8_SUFFIX.get(dtype)
    # one test on the common path; the checks that name what is wrong run where it fails
    if not (len(zshape) == 2 and len(wshape) == 3 and z.dtype is torch.int8 and weights_q.dtype is torch.int8
            and wshape[2] == zshape[1] and wshape[0] == p and 1 <= p <= 4 and zshape[0] <= MAX_ROWS and z_scale.shape == zshape[:1]
            and weights_scale.shape == wshape[:2] and z_scale.dtype is torch.float32
            and weights_scale.dtype is torch.float32 and device >= 0 and z_scale.get_device() == device
            and weights_q.get_device() == device and weights_scale.get_device() == device
            and min(used) >= 1 and max(used) <= wshape[1] <= MAX_ROWS and zshape[1] & 15 == 0 and 16 <= zshape[1] <= 16384
            and suffix is not None and (sigmoid_block is None or 0 <= sigmoid_block < p)
            and not (z_scale.requires_grad or weights_scale.requires_grad)):
        _check_projection_int8(z, z_scale, weights_q, weights_scale, used, sigmoid_block, dtype)
    m, d = zshape
    zc, wc, zs, ws, on = _aligned(z), _aligned(weights_q), z_scale.contiguous(), weights_scale.contiguous(), z.device
    outs = [torch.empty((m, u), dtype=dtype, device=on) for u in used]
    ptrs = [o.data_ptr() for o in outs] + [0] * (4 - p)
    widths = [*used] + [1] * (4 - p)
    with _lib.on_device(on):
        _lib.call(f"vsp_project_int8_{suffix}", zc.data_ptr(), zs.data_ptr(), wc.data_ptr(), ws.data_ptr(), p, wshape[1], d,
                  m, *widths, *ptrs, -1 if sigmoid_block is None else sigmoid_block, _lib.stream_of(on))
    return outs


def _check_projection_int8(z: Tensor, z_scale: Tensor, weights_q: Tensor, weights_scale: Tensor, used: tuple[int, ...],
                           sigmoid_block: int | None, dtype: torch.dtype) -> None:
    """Raises for what ``projection_int8`` does not take."""
    if weights_q.dim() == 3 and weights_q.shape[1] > MAX_ROWS:
        raise ContractError(f"weights_q: {weights_q.shape[1]} columns, the kernel takes at most {MAX_ROWS}")
    if z.dim() != 2 or z.dtype != torch.int8 or z.device.type != "cuda":
        raise ContractError(f"z: int8 [M, d] on CUDA, got {tuple(z.shape)} {z.dtype} on {z.device}")
    m, d = z.shape
    if weights_q.dim() != 3 or weights_q.dtype != torch.int8 or weights_q.shape[2] != d:
        raise ContractError(f"weights_q: int8 [p, cols, {d}], got {tuple(weights_q.shape)} {weights_q.dtype}")
    p, cols = weights_q.shape[0], weights_q.shape[1]
    for name, t, shape in (("z_scale", z_scale, (m,)), ("weights_scale", weights_scale, (p, cols))):
        if t.shape != shape or t.dtype != torch.float32:
            raise ContractError(f"{name}: float32 {shape}, got {tuple(t.shape)} {t.dtype}")
    for name, t in (("z_scale", z_scale), ("weights_q", weights_q), ("weights_scale", weights_scale)):
        if t.device != z.device:
            raise ContractError(f"{name} is on {t.device}, z on {z.device}")
    if len(used) != p or not 1 <= p <= 4 or any(not 1 <= u <= cols for u in used):
        raise ContractError(f"used: {p} widths in 1..{cols}, got {tuple(used)}")
    if m > MAX_ROWS:
        raise ContractError(f"z: {m} rows, the kernel takes at most {MAX_ROWS}")
    if d % 16 or not 16 <= d <= 16384:
        raise ContractError(f"z: width {d} is not a multiple of 16 in 16..16384")
    if sigmoid_block is not None and not 0 <= sigmoid_block < p:
        raise ContractError(f"sigmoid_block {sigmoid_block} is not one of the {p} blocks")
    if dtype not in _INT8_SUFFIX:
        raise ContractError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
    _refuse_grad("projection_int8", z_scale, weights_scale)
