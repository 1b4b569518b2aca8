"""The gated delta rule on MI355X: the delta rule of ``delta_scan`` with a decay of the state before each token.

Per head the state ``H [dk, dk]`` (key rows, value columns, float32) and per token the log decay ``g``:

    ``H_t = e^{g_t} H_{t-1} + k_t u_t^T``, ``u_t = beta_t (v_t - e^{g_t} H_{t-1}^T k_t)``, ``o_t = H_t^T q_t``

With ``g = 0`` it is the delta rule of ``delta_scan_fused`` (``vesper/recurrence.py:118-163``), whose layouts, checks
and ``active`` mask these functions share: no query scaling, keys already normalised.

- ``gated_delta_scan``: a block of tokens, chunked, with its backward pass (``vsp_gated_scan_*``).
- ``gated_delta_step``: one token per row, for decoding (``vsp_gated_step_*``), forward only.

bfloat16 inputs run bf16 MFMA, with everything that is computed in float32 and multiplied again as the sum of three
bf16 numbers (24 bits; in the outputs' products two): the states and the decays' gradients come out as exact as float32 sums
give them, the latter behind strong decays too (every term of a decay's gradient carries that decay).
float32 inputs run float32 MFMA.
"""

from __future__ import annotations

import functools
from typing import Any

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from vesper.contracts import ContractError, Dims, check_shape, refuse_tangents
from vesper.kernels import _lib
from vesper.kernels.delta_scan import MAX_HEAD_DIM, STATE_DTYPE, _active_mask, _aligned, _refuse_grad

GATE_DTYPE = torch.float32  # the log decays: sums of many of them decide what is left of a state
INPUT_DTYPES = (torch.bfloat16, torch.float32)  # of q, k, v and beta, all alike
MAX_TOKENS = 2**30  # of a row
MAX_FEATURES = 2**22  # of a token's heads, a head's rounded up to a multiple of 8
MAX_CHUNKS = 2**25  # of 64 tokens, over all rows and heads
MAX_KEPT_CHUNKS = 2**23 - 1  # where the backward follows: 512 threads each
MAX_SLICES = 2**22  # of 16 value columns, over all rows and heads
MAX_STEP_HEADS = 2**20 - 1  # rows times heads of one launch of the step
_SUFFIX = {torch.bfloat16: "bf16", torch.float32: "f32"}
_STEP = {dtype: f"vsp_gated_step_{suffix}" for dtype, suffix in _SUFFIX.items()}
_SCAN = {dtype: f"vsp_gated_scan_{suffix}" for dtype, suffix in _SUFFIX.items()}
_SCAN_BACKWARD = {dtype: f"vsp_gated_scan_backward_{suffix}" for dtype, suffix in _SUFFIX.items()}


@functools.lru_cache(maxsize=256)
def _bytes(what: str, *sizes: int) -> int:
    """A size that the library gives for sizes: the workspaces' and the records'."""
    return int(getattr(_lib.library(), f"vsp_gated_scan_{what}_bytes")(*sizes))


def _check(q: Tensor, k: Tensor, v: Tensor, beta: Tensor, g: Tensor, state: Tensor, lead: tuple[str, ...]) -> Dims:
    """Shapes, dtypes, devices and the width, with the error texts of ``delta_scan``'s checks: one comparison each for what is
    in order (1.6 us against 3.3 for a call whose kernel takes 4), and what is not is looked for one by one."""
    shape, dtype, device = q.shape, q.dtype, q.device
    if (len(shape) == len(lead) + 1 and k.shape == shape == v.shape and beta.shape == g.shape == shape[:-1]
            and state.shape == (shape[0], shape[-2], shape[-1], shape[-1]) and dtype in _SUFFIX
            and dtype is k.dtype is v.dtype is beta.dtype and g.dtype is GATE_DTYPE and state.dtype is STATE_DTYPE
            and device == k.device == v.device == beta.device == g.device == state.device and device.type == "cuda"
            and 1 <= shape[-1] <= MAX_HEAD_DIM):
        return dict(zip((*lead, "dk"), shape))
    if dtype not in INPUT_DTYPES:
        raise ContractError(f"q: dtype must be torch.bfloat16 or torch.float32, got {dtype}")
    dims: Dims = {}
    for name, t in (("q", q), ("k", k), ("v", v)):
        check_shape(name, t, (*lead, "dk"), dims, dtype)
    check_shape("beta", beta, lead, dims, dtype)
    check_shape("g", g, lead, dims, GATE_DTYPE)
    check_shape("state", state, ("b", "h", "dk", "dk"), dims, STATE_DTYPE)
    if q.device.type != "cuda":
        raise ContractError(f"the fused scan runs on CUDA only, got q on {q.device}")
    for name, t in (("k", k), ("v", v), ("beta", beta), ("g", g), ("state", state)):
        if t.device != q.device:
            raise ContractError(f"{name} is on {t.device}, q on {q.device}")
    if not 1 <= dims["dk"] <= MAX_HEAD_DIM:
        raise ContractError(f"head dimension {dims['dk']} exceeds the kernel's {MAX_HEAD_DIM}" if dims["dk"]
                            else "head dimension 0: the kernel takes 1 and more")
    return dims


def _check_sizes(b: int, n: int, h: int, dk: int, grad: bool) -> None:
    """Raises for sizes past the kernels' launches and offsets (what the C entries count in 32 bits among them)."""
    chunks, slices = b * h * -(-n // 64), b * h * -(-dk // 16)
    if (n <= MAX_TOKENS and h * dk <= MAX_FEATURES - 7 * h and chunks <= (MAX_KEPT_CHUNKS if grad else MAX_CHUNKS)
            and slices <= MAX_SLICES):
        return
    if n > MAX_TOKENS:
        raise ContractError(f"q: {n} tokens a row, the kernels take at most 2**30")
    if h * (dk + -dk % 8) > MAX_FEATURES:
        raise ContractError(f"q: {h} heads of {dk + -dk % 8} features a token, the kernels take at most 2**22 features")
    if chunks > MAX_CHUNKS or (grad and chunks > MAX_KEPT_CHUNKS):
        most = "2**23 - 1 under autograd" if grad else "2**25"
        raise ContractError(f"q: {chunks} chunks of 64 tokens over all rows and heads, the kernels take at most {most}")
    if slices > MAX_SLICES:
        raise ContractError(f"q: {slices} slices of 16 value columns over all rows and heads, the kernels take at most 2**22")


def _forward(q: Tensor, k: Tensor, v: Tensor, beta: Tensor, g: Tensor, state: Tensor, mask: Tensor | None,
             records: Tensor | None) -> tuple[Tensor, Tensor]:
    """The scan of contiguous, aligned tensors at a width that is a multiple of 8."""
    b, n, h, dk = q.shape
    o, s_out = torch.empty_like(q), torch.empty_like(state)
    ws_bytes = _bytes("workspace", b, n, h, dk, int(q.dtype == torch.float32))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    _lib.launch(q.device, _SCAN[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), beta.data_ptr(), g.data_ptr(),
                state.data_ptr(), o.data_ptr(), s_out.data_ptr(), ws.data_ptr(), ws_bytes,
                None if records is None else records.data_ptr(), 0 if records is None else records.numel(),
                None if mask is None else mask.data_ptr(), b, n, h, dk)
    return o, s_out


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, q: Tensor, k: Tensor, v: Tensor, beta: Tensor, g: Tensor, state: Tensor,
                mask: Tensor | None) -> tuple[Tensor, Tensor]:  # noqa: D102
        ctx.set_materialize_grads(False)
        q, k, v, beta, g, state = _aligned(q), _aligned(k), _aligned(v), _aligned(beta), _aligned(g), _aligned(state)
        # each chunk's starting state and its Delta, for the backward
        records = torch.empty(_bytes("records", *q.shape), dtype=torch.uint8, device=q.device)
        o, s_out = _forward(q, k, v, beta, g, state, mask, records)
        if mask is None:
            ctx.save_for_backward(q, k, v, beta, g, records)
        else:
            ctx.save_for_backward(q, k, v, beta, g, records, mask)
        return o, s_out

    @staticmethod
    def backward(ctx: Any, d_o: Tensor | None, d_state: Tensor | None) -> tuple[Tensor | None, ...]:  # noqa: D102
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, d_o, d_state)


def _backward(ctx: Any, d_o: Tensor | None, d_state: Tensor | None) -> tuple[Tensor | None, ...]:
    q, k, v, beta, g, records, *rest = ctx.saved_tensors
    b, n, h, dk = q.shape
    go = torch.zeros_like(q) if d_o is None else _aligned(d_o.to(q.dtype))
    gs = None if d_state is None else _aligned(d_state.to(STATE_DTYPE))
    dq, dk_, dv, db, dg = (torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(beta),
                           torch.empty_like(g))
    d_state_in = torch.empty((b, h, dk, dk), dtype=STATE_DTYPE, device=q.device)
    ws_bytes = _bytes("backward_workspace", b, n, h, dk, int(q.dtype == torch.float32))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    _lib.launch(q.device, _SCAN_BACKWARD[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), beta.data_ptr(), g.data_ptr(),
                records.data_ptr(), records.numel(), go.data_ptr(), None if gs is None else gs.data_ptr(),
                rest[0].data_ptr() if rest else None, dq.data_ptr(), dk_.data_ptr(), dv.data_ptr(), db.data_ptr(),
                dg.data_ptr(), d_state_in.data_ptr(), ws.data_ptr(), ws_bytes, b, n, h, dk)
    need = ctx.needs_input_grad
    if all(need[:6]):
        return dq, dk_, dv, db, dg, d_state_in, None
    return (*(x if wanted else None for x, wanted in zip((dq, dk_, dv, db, dg, d_state_in), need)), None)


_backward_once = once_differentiable(_backward)  # under create_graph: its results refuse a derivative


def gated_delta_scan(q: Tensor, k: Tensor, v: Tensor, beta: Tensor, g: Tensor, state: Tensor, *,
                     active: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """The gated delta rule over a block of ``n`` tokens (chunks of 64, float32 state).

    Args:
        q: the queries ``[b, n, h, dk]``, bfloat16 or float32, on the GPU; ``dk`` in 1..256.
        k: the keys, same shape and dtype; the caller normalizes them (norm at most one).
        v: the values, same shape and dtype.
        beta: the write strengths ``[b, n, h]``, same dtype, each in [0, 1].
        g: the log decays ``[b, n, h]``, float32, each at most 0; ``-inf`` forgets the state (the start of a
            document in a packed row) and gives its log decay a gradient of 0.
        state: the float32 state ``[b, h, dk, dk]`` the block starts from.
        active: optional bool ``[b, n]``: a token marked False still decays and updates the state, but its output
            row is zero.

    Returns:
        ``(o, state_n)``: the outputs ``[b, n, h, dk]`` in q's dtype and the float32 state after the block; for
        ``n == 0`` the (empty) ``q`` tensor itself and the same ``state`` object.

    Under autograd the gradients of ``q, k, v, beta, g`` and ``state`` come from the backward kernels; the forward
    then keeps each chunk's starting state and corrections, ``4 w (w + 64)`` bytes a chunk and head, ``w`` being ``dk`` rounded
    up to a multiple of 16. Widths that
    are no multiple of 8 run zero-padded to the next, which changes no output. One token without autograd runs as
    ``gated_delta_step``. The backward may be captured into a graph, as long as no eager graph of the same leaves is alive
    (torch's accumulation into them would leave the capture). A NaN or an infinity in a token reaches its head's outputs from the start of its chunk on (a
    chunk's products are over all pairs of its tokens), not those of other heads and rows.

    At most ``2**30`` tokens a row, ``2**22`` features a token (a head's rounded up to a multiple of 8), ``2**25`` chunks of 64
    tokens (``2**23 - 1`` under autograd) and ``2**22`` slices of 16 value columns over all rows and heads.

    Raises:
        ContractError: on a dtype, shape, device, width or size outside the contract or a forward-mode tangent, before any
            kernel runs.
    """
    dims = _check(q, k, v, beta, g, state, ("b", "n", "h"))
    if forward_ad._current_level >= 0:  # noqa: SLF001
        refuse_tangents(q, k, v, beta, g, state)
    if active is not None:
        check_shape("active", active, ("b", "n"), dims, torch.bool)
    if dims["n"] == 0:
        return q, state
    mask = None if active is None else _active_mask(active, ("b", "n"), dims, q.device)
    if dims["b"] == 0 or dims["h"] == 0:  # empty results that keep the graph
        o = q + k + v + (beta + g.to(q.dtype))[..., None] + state.sum().to(q.dtype)
        return o, state + o.sum().to(STATE_DTYPE)
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or beta.requires_grad
                                        or g.requires_grad or state.requires_grad)
    dk = dims["dk"]
    if dims["n"] == 1 and not grad:
        first = (t[:, 0] for t in (q, k, v, beta, g))
        o, after = gated_delta_step(*first, state.contiguous(), active=None if active is None else active[:, 0])
        return o[:, None], after
    _check_sizes(dims["b"], dims["n"], dims["h"], dk, grad)
    pad = -dk % 8
    if pad:
        q, k, v = (torch.nn.functional.pad(t, (0, pad)) for t in (q, k, v))
        state = torch.nn.functional.pad(state, (0, pad, 0, pad))
    if grad:
        o, after = _GatedScan.apply(q, k, v, beta, g, state, mask)
    else:
        o, after = _forward(_aligned(q), _aligned(k), _aligned(v), _aligned(beta), _aligned(g), _aligned(state), mask, None)
    return (o[..., :dk].contiguous(), after[..., :dk, :dk].contiguous()) if pad else (o, after)


def gated_delta_step(q: Tensor, k: Tensor, v: Tensor, beta: Tensor, g: Tensor, state: Tensor, *,
                     active: Tensor | None = None, out_state: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """One token per row through the gated delta rule, decayed, written, then read: ``(H'^T q, H')``.

    Args:
        q, k, v: ``[b, h, dk]`` float32 or bfloat16 (all three alike, ``beta [b, h]`` too), ``dk`` in 1..256, ``h`` under
            ``2**20`` (rows of as many heads in all run in one launch, more in several).
        g: the log decays ``[b, h]``, float32.
        state: ``[b, h, dk, dk]`` float32, contiguous.
        active: optional bool ``[b]``; an inactive row decays and writes the state and reads zero.
        out_state: optional contiguous float32 tensor shaped like ``state`` that receives the new state; it may be
            ``state`` itself (an in-place decode step), and overlaps it and the other inputs in no other way.

    Returns:
        ``(o [b, h, dk], state')`` with ``o`` in the inputs' dtype.

    Raises:
        ContractError: on a dtype, shape, device or width outside the contract, or inputs that require a gradient
            while grad mode is on.
    """
    dims = _check(q, k, v, beta, g, state, ("b", "h"))
    if forward_ad._current_level >= 0:  # noqa: SLF001
        refuse_tangents(q, k, v, beta, g, state)
    if torch.is_grad_enabled():
        _refuse_grad(q, k, v, beta, g, state)
    b, h, dk = q.shape
    if h > MAX_STEP_HEADS:
        raise ContractError(f"q: {h} heads, the step takes at most 2**20 - 1")
    if not state.is_contiguous():
        raise ContractError("state must be contiguous")
    given = out_state is not None
    if out_state is None:
        out_state = torch.empty_like(state)
    elif out_state is not state:
        check_shape("out_state", out_state, ("b", "h", "dk", "dk"), dims, STATE_DTYPE)
        if out_state.device != q.device or not out_state.is_contiguous():
            raise ContractError("out_state must be a contiguous tensor on q's device")
        if out_state.requires_grad and torch.is_grad_enabled():
            raise ContractError("out_state must not require a gradient: the step writes it in place")
        if 0 < abs(out_state.data_ptr() - state.data_ptr()) < state.nbytes:
            raise ContractError("out_state must be state itself or not overlap it")
    q, k, v, beta, g = q.contiguous(), k.contiguous(), v.contiguous(), beta.contiguous(), g.contiguous()
    mask = None if active is None else _active_mask(active, ("b",), dims, q.device)
    o = torch.empty_like(q)
    if b == 0 or h == 0:
        return o, out_state
    qp, kp, vp, bp, gp, to = q.data_ptr(), k.data_ptr(), v.data_ptr(), beta.data_ptr(), g.data_ptr(), out_state.data_ptr()
    if given:  # a workgroup would write what others are yet to read
        strength = (2 if q.dtype is torch.bfloat16 else 4) * b * h  # bytes of beta; of q, k and v dk times as many
        behind, token = to + 4 * b * h * dk * dk, strength * dk
        if ((qp < behind and to < qp + token) or (kp < behind and to < kp + token) or (vp < behind and to < vp + token)
                or (bp < behind and to < bp + strength) or (gp < behind and to < gp + 4 * b * h)):
            raise ContractError("out_state must not overlap q, k, v, beta or g")
    if b * h <= MAX_STEP_HEADS:
        _lib.launch(q.device, _STEP[q.dtype], qp, kp, vp, bp, gp, state.data_ptr(), to, o.data_ptr(),
                    None if mask is None else mask.data_ptr(), b, h, dk)
        return o, out_state
    rows = MAX_STEP_HEADS // h
    for i in range(0, b, rows):
        part = [t[i : i + rows] for t in (q, k, v, beta, g, state, out_state, o, *(() if mask is None else (mask,)))]
        _lib.launch(q.device, _STEP[q.dtype], *(t.data_ptr() for t in part), *(() if mask is not None else (None,)),
                    part[0].shape[0], h, dk)
    return o, out_state
