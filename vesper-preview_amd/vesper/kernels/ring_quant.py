"""The decoder's KV ring held in four bits, on MI355X (HIP kernels through the C ABI).

``QuantRingKVCache`` is ``RingKVCache`` (``vesper/kernels/ring_attn.py``) in a quarter of the memory: a
token at position ``p`` lives in slot ``p % window``, ``pos`` and ``valid`` say what a slot holds, and a
row of keys or values (one token, one KV head) is ``dk`` codes of four bits with one pair of scale and
minimum:

    scale = (max - min) / 15 rounded to the cache's dtype, code = round((x - min) / scale) in 0..15,
    value = min + scale * code

so a row takes ``dk / 2 + 4`` bytes in place of ``2 dk``. Rows are held head by head (``k [b, hkv, window,
dk / 2]``): a head's rows are contiguous for the workgroup that attends them.

- ``quant_ring_write``: a chunk of tokens (a prompt, a padded batch of prompts) quantised into its slots;
- ``quant_ring_read``: tokens read back by position, as the chunk attention's ``KVCache`` rows;
- ``quant_ring_attention``: one new token per row over the ring and itself, then written into its slot,
  the counterpart of ``ring_attention`` (``WindowedAttention.attend_ring``, ``vesper/attention.py:298-338``,
  and ``kv_ring_write``, ``:104-139``).

All are forward only.
"""

from __future__ import annotations

import functools
import math
from dataclasses import dataclass

import torch
from torch import Tensor

from vesper.contracts import ContractError, Dims, check_shape, require
from vesper.kernels import _lib
from vesper.kernels.ring_attn import MAX_GROUP, MAX_HEAD_DIM, _aligned

MAX_KV_HEADS = 16384  # a workgroup's tokens are addressed by 32-bit offsets
MAX_COUNT = 2**31 - 1  # rows, tokens a row and slots: the C entries count each in 32 bits
_SUFFIX = {torch.bfloat16: "bf16", torch.float16: "f16"}


@dataclass(frozen=True)
class QuantRingKVCache:
    """A decoding window of ``window`` slots in four bits; slot order is not age order.

    ``k``, ``v`` uint8 ``[b, hkv, window, dk / 2]`` (feature ``2 i`` in the low half of byte ``i``);
    ``k_scale``, ``v_scale`` bfloat16 or float16 ``[b, hkv, window, 2]`` (scale, minimum); ``pos`` int64 and
    ``valid`` bool ``[b, window]``.
    """

    k: Tensor
    v: Tensor
    k_scale: Tensor
    v_scale: Tensor
    pos: Tensor
    valid: Tensor
    window: int

    def tensors(self) -> tuple[Tensor, ...]:
        return self.k, self.v, self.k_scale, self.v_scale, self.pos, self.valid


def quant_ring_empty(b: int, hkv: int, dk: int, window: int, dtype: torch.dtype, device: torch.device) -> QuantRingKVCache:
    """Every slot unwritten: zero codes, scales and minima, positions 0, ``valid`` False. ``dtype`` is that of
    the tokens (bfloat16 or float16).

    Raises:
        ValueError: if ``window`` is below 1; ContractError: on a size, head width or dtype outside the contract.
    """
    if window < 1:
        raise ValueError(f"window must be at least 1, got {window}")
    _check_counts({"b": b, "w": window})
    _check_width(dk)
    if dtype not in _SUFFIX:
        raise ContractError(f"the ring's dtype must be bfloat16 or float16, got {dtype}")
    codes = (b, hkv, window, dk // 2)
    return QuantRingKVCache(
        k=torch.zeros(codes, dtype=torch.uint8, device=device),
        v=torch.zeros(codes, dtype=torch.uint8, device=device),
        k_scale=torch.zeros(b, hkv, window, 2, dtype=dtype, device=device),
        v_scale=torch.zeros(b, hkv, window, 2, dtype=dtype, device=device),
        pos=torch.zeros(b, window, dtype=torch.long, device=device),
        valid=torch.zeros(b, window, dtype=torch.bool, device=device),
        window=window,
    )


def _check_width(dk: int) -> None:
    if dk % 8 != 0 or not 8 <= dk <= MAX_HEAD_DIM:
        raise ContractError(f"head dimension {dk}: the kernels take multiples of 8 up to {MAX_HEAD_DIM}")


def _check_counts(dims: Dims) -> None:
    for name, what in (("b", "rows"), ("n", "tokens a row"), ("w", "slots")):
        if dims.get(name, 0) > MAX_COUNT:
            raise ContractError(f"{dims[name]} {what}, the kernels take at most {MAX_COUNT}")


def _check_ring(cache: QuantRingKVCache, dims: Dims) -> torch.dtype:
    """The ring's shapes, sizes and dtypes under ``dims``; its tokens' dtype."""
    dims["w"], dims["pair"] = cache.window, 2
    check_shape("cache.k", cache.k, ("b", "hkv", "w", "half"), dims, torch.uint8)
    check_shape("cache.v", cache.v, ("b", "hkv", "w", "half"), dims, torch.uint8)
    check_shape("cache.k_scale", cache.k_scale, ("b", "hkv", "w", "pair"), dims)
    check_shape("cache.v_scale", cache.v_scale, ("b", "hkv", "w", "pair"), dims, cache.k_scale.dtype)
    check_shape("cache.pos", cache.pos, ("b", "w"), dims, torch.long)
    check_shape("cache.valid", cache.valid, ("b", "w"), dims, torch.bool)
    _check_counts(dims)
    dtype = cache.k_scale.dtype
    _refuse_grad(cache.k_scale, cache.v_scale)
    if dtype not in _SUFFIX:
        raise ContractError(f"cache.k_scale: dtype must be bfloat16 or float16, got {dtype}")
    if cache.window < 1:
        raise ContractError(f"the ring's window must be at least 1, got {cache.window}")
    if dims["hkv"] > MAX_KV_HEADS:
        raise ContractError(f"cache.k: {dims['hkv']} KV heads, the kernels take at most {MAX_KV_HEADS}")
    dk = 2 * dims["half"]
    if dims.setdefault("dk", dk) != dk:
        raise ContractError(f"cache.k: rows of {dims['half']} bytes hold {dk} features, the tokens have {dims['dk']}")
    _check_width(dk)
    return dtype


def _check_devices(cache: QuantRingKVCache, first: str, device: torch.device, *named: tuple[str, Tensor]) -> None:
    if device.type != "cuda":
        raise ContractError(f"the four-bit ring's kernels run on CUDA only, got {first} on {device}")
    for name, t in (*named, ("cache.k", cache.k), ("cache.v", cache.v), ("cache.k_scale", cache.k_scale),
                    ("cache.v_scale", cache.v_scale), ("cache.pos", cache.pos), ("cache.valid", cache.valid)):
        if t.device != device:
            raise ContractError(f"{name} is on {t.device}, {first} on {device}")


def _ring_as_is(cache: QuantRingKVCache, b: int, hkv: int, dk: int, dtype: torch.dtype, device: int) -> bool:
    """Whether every tensor of the ring is what the kernels take as it is: one test on the common path in place of
    the checks that name what is wrong (a decode step's call spends more on those than its kernel runs)."""
    w, k, v, ks, vs, pos, valid = cache.window, cache.k, cache.v, cache.k_scale, cache.v_scale, cache.pos, cache.valid
    codes, pairs, slots = (b, hkv, w, dk >> 1), (b, hkv, w, 2), (b, w)
    return (k.shape == codes and v.shape == codes and ks.shape == pairs and vs.shape == pairs
            and pos.shape == slots and valid.shape == slots
            and k.dtype is torch.uint8 and v.dtype is torch.uint8 and ks.dtype is dtype and vs.dtype is dtype
            and pos.dtype is torch.int64 and valid.dtype is torch.bool
            and k.get_device() == device and v.get_device() == device and ks.get_device() == device
            and vs.get_device() == device and pos.get_device() == device and valid.get_device() == device
            and k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()
            and pos.is_contiguous() and valid.is_contiguous()
            and (k.data_ptr() | v.data_ptr() | ks.data_ptr() | vs.data_ptr()) & 3 == 0
            and not (ks.requires_grad or vs.requires_grad)
            and 1 <= w <= MAX_COUNT and b <= MAX_COUNT
            and dk & 7 == 0 and 8 <= dk <= MAX_HEAD_DIM and 1 <= hkv <= MAX_KV_HEADS)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(b: int, h: int, hkv: int, dk: int, w: int) -> int:
    return int(_lib.library().vsp_quant_ring_attn_workspace_bytes(b, h, hkv, dk, w))


def _writable(cache: QuantRingKVCache, inplace: bool) -> QuantRingKVCache:
    """The ring that a kernel writes: the cache's own tensors, or a contiguous copy."""
    if not inplace:
        return QuantRingKVCache(*(t.clone(memory_format=torch.contiguous_format) for t in cache.tensors()), cache.window)
    for name, t in zip(("k", "v", "k_scale", "v_scale", "pos", "valid"), cache.tensors()):
        if not t.is_contiguous():
            raise ContractError(f"cache.{name} must be contiguous for an in-place ring")
        if t.data_ptr() % 4 != 0 and name not in ("pos", "valid"):
            raise ContractError(f"cache.{name} must be 4-byte aligned for an in-place ring")
    return cache


def _refuse_grad(*tensors: Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ContractError("the four-bit ring is forward only: call it under torch.no_grad()")


def quant_ring_write(k: Tensor, v: Tensor, pos: Tensor, cache: QuantRingKVCache, *, lengths: Tensor | None = None,
                     inplace: bool = False, check_positions: bool = True) -> QuantRingKVCache:
    """A chunk of tokens quantised into the ring (``vsp_quant_ring_write_*``, one launch).

    Args:
        k, v: ``[b, n, hkv, dk]`` rotated keys and values in the ring's dtype.
        pos: ``[b, n]`` int64 nonnegative positions, going up by one along each row (the kernel reads some of
            a row's and counts on from them).
        cache: the ring; a row's last ``window`` tokens replace what their slots hold.
        lengths: optional int32 or int64 ``[b]``, 0 to ``n``: row ``i`` writes its first ``lengths[i]`` tokens only (a
            padded batch); the others, and their positions, are not looked at.
        inplace: write into ``cache``'s tensors instead of a copy.
        check_positions: hold the contract of ``pos`` and ``lengths`` with ``require`` (a device assert under
            graph capture).

    Returns:
        the ring that holds the tokens (``cache`` itself when ``inplace``).

    Raises:
        ContractError: on shapes, dtypes, devices or values outside that contract.
    """
    shape, dtype, device, w = k.shape, k.dtype, k.get_device(), cache.window
    as_is = (len(shape) == 4 and v.shape == shape and shape[1] <= MAX_COUNT and pos.shape == shape[:2] and v.dtype is dtype
             and pos.dtype is torch.int64 and dtype in _SUFFIX and device >= 0 and v.get_device() == device
             and pos.get_device() == device and not (k.requires_grad or v.requires_grad)
             and _ring_as_is(cache, shape[0], shape[2], shape[3], dtype, device))
    if not as_is:
        dims: Dims = {}
        check_shape("k", k, ("b", "n", "hkv", "dk"), dims)
        check_shape("v", v, ("b", "n", "hkv", "dk"), dims, k.dtype)
        check_shape("pos", pos, ("b", "n"), dims, torch.long)
        if _check_ring(cache, dims) != dtype:
            raise ContractError(f"k: dtype must be the ring's {cache.k_scale.dtype}, got {dtype}")
        _check_devices(cache, "k", k.device, ("v", v), ("pos", pos))
        _refuse_grad(k, v)
    b, n, hkv, dk = shape
    if lengths is not None:
        check_shape("lengths", lengths, (b,), {})
        if lengths.dtype not in (torch.int32, torch.long):
            raise ContractError(f"lengths: dtype must be int32 or int64, got {lengths.dtype}")
        if lengths.device != k.device:
            raise ContractError(f"lengths is on {lengths.device}, k on {k.device}")
    if check_positions and b > 0 and n > 0:
        ok = (pos[:, 1:] - pos[:, :-1] == 1)
        first = pos[:, 0] >= 0
        if lengths is not None:
            ok = ok | (torch.arange(1, n, device=pos.device) >= lengths[:, None])
            first = (first | (lengths == 0)) & (lengths >= 0) & (lengths <= n)
        require((ok.all() & first.all()).reshape(1),
                "quant_ring_write: positions must be nonnegative and consecutive, lengths in 0..n")
    ring = cache if inplace and as_is else _writable(cache, inplace)
    if b == 0 or n == 0:
        return ring
    if lengths is not None:
        lengths = lengths.long().contiguous()
    k, v, pos, on = _aligned(k), _aligned(v), pos.contiguous(), k.device
    with _lib.on_device(on):
        _lib.call(f"vsp_quant_ring_write_{_SUFFIX[dtype]}", k.data_ptr(), v.data_ptr(), pos.data_ptr(),
                  _lib.ptr(lengths), ring.k.data_ptr(), ring.v.data_ptr(), ring.k_scale.data_ptr(),
                  ring.v_scale.data_ptr(), ring.pos.data_ptr(), ring.valid.data_ptr(), b, n, hkv, dk, w,
                  _lib.stream_of(on))
    return ring


def quant_ring_read(cache: QuantRingKVCache, pos: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """Tokens of the ring by position (``vsp_quant_ring_read_*``, one launch): ``(k, v, found)``.

    Args:
        cache: the ring.
        pos: ``[b, n]`` int64 positions, in any order, any of them more than once.

    Returns:
        ``k, v [b, n, hkv, dk]`` in the ring's dtype and ``found [b, n]`` bool: where the ring does not hold
        the position (never written, replaced since, or negative) ``found`` is False and the rows are zero.

    Raises:
        ContractError: on shapes, dtypes or devices outside that contract.
    """
    dtype, shape, device = cache.k_scale.dtype, cache.k.shape, pos.get_device()
    held = cache
    if not (len(shape) == 4 and pos.dim() == 2 and pos.shape[0] == shape[0] and pos.shape[1] <= MAX_COUNT
            and pos.dtype is torch.int64 and dtype in _SUFFIX and device >= 0
            and _ring_as_is(cache, shape[0], shape[1], 2 * shape[3], dtype, device)):
        dims: Dims = {}
        check_shape("pos", pos, ("b", "n"), dims, torch.long)
        _check_ring(cache, dims)
        _check_devices(cache, "pos", pos.device)
        parts = [t.contiguous() for t in cache.tensors()]
        held = QuantRingKVCache(*(t if t.data_ptr() % 4 == 0 or t.dtype == torch.bool else t.clone() for t in parts),
                                cache.window)
    (b, n), hkv, dk, on = pos.shape, shape[1], 2 * shape[3], pos.device
    k = torch.empty((b, n, hkv, dk), dtype=dtype, device=on)
    v = torch.empty_like(k)
    found = torch.empty((b, n), dtype=torch.bool, device=on)
    if b == 0 or n == 0:
        return k, v, found
    pos = pos.contiguous()
    with _lib.on_device(on):
        _lib.call(f"vsp_quant_ring_read_{_SUFFIX[dtype]}", held.k.data_ptr(), held.v.data_ptr(), held.k_scale.data_ptr(),
                  held.v_scale.data_ptr(), held.pos.data_ptr(), held.valid.data_ptr(), pos.data_ptr(), k.data_ptr(),
                  v.data_ptr(), found.data_ptr(), b, n, hkv, dk, cache.window, _lib.stream_of(on))
    return k, v, found


def quant_ring_attention(q: Tensor, k: Tensor, v: Tensor, pos: Tensor, cache: QuantRingKVCache, *,
                         active: Tensor | None = None, inplace: bool = False,
                         check_positions: bool = True) -> tuple[Tensor, QuantRingKVCache]:
    """One new token per row over the four-bit ring and itself; then the token is quantised into its slot
    (``vsp_quant_ring_attn_*``: one launch, and one more that joins the parts where a window is shared by
    several workgroups).

    The query at position ``p`` attends the valid slots with positions in ``(p - window, p]`` other than slot
    ``p % window`` (which the new token replaces; in a ring in use it holds position ``p - window`` or
    nothing), and the new token once, from its argument. A ring that already holds position ``p`` (a step
    repeated) therefore gives the same result again, unlike ``ring_attention``'s, which attends such a slot too.

    Args:
        q: ``[b, 1, h, dk]`` rotated queries in the ring's dtype; at most 8 query heads a KV head.
        k, v: ``[b, 1, hkv, dk]`` the new token's rotated key and value.
        pos: ``[b, 1]`` int64 nonnegative positions.
        cache: the ring.
        active: optional bool ``[b]``; an inactive row's output is zero, its token is still written.
        inplace: write into ``cache``'s tensors instead of a copy.
        check_positions: hold ``pos >= 0`` with ``require`` (a device assert under graph capture).

    Returns:
        ``(o [b, 1, h, dk], ring)`` with the ring that holds the new tokens.

    Raises:
        ContractError: on shapes, dtypes, devices or values outside that contract.
    """
    shape, new, dtype, device, w = q.shape, k.shape, q.dtype, q.get_device(), cache.window
    as_is = (len(shape) == 4 and len(new) == 4 and shape[1] == 1 and new[1] == 1 and new[0] == shape[0]
             and new[3] == shape[3] and v.shape == new and pos.shape == shape[:2] and k.dtype is dtype
             and v.dtype is dtype and pos.dtype is torch.int64 and dtype in _SUFFIX and device >= 0
             and k.get_device() == device and v.get_device() == device and pos.get_device() == device
             and not (q.requires_grad or k.requires_grad or v.requires_grad)
             and _ring_as_is(cache, shape[0], new[2], shape[3], dtype, device))
    if not as_is:
        dims: Dims = {"one": 1}
        check_shape("q", q, ("b", "one", "h", "dk"), dims)
        check_shape("k", k, ("b", "one", "hkv", "dk"), dims, dtype)
        check_shape("v", v, ("b", "one", "hkv", "dk"), dims, dtype)
        check_shape("pos", pos, ("b", "one"), dims, torch.long)
        if _check_ring(cache, dims) != dtype:
            raise ContractError(f"q: dtype must be the ring's {cache.k_scale.dtype}, got {dtype}")
        _check_devices(cache, "q", q.device, ("k", k), ("v", v), ("pos", pos))
        _refuse_grad(q, k, v)
    b, h, hkv, dk = shape[0], shape[2], new[2], shape[3]
    if hkv < 1 or h < 1 or h % hkv != 0 or h // hkv > MAX_GROUP:
        raise ContractError(f"{h} query heads over {hkv} KV heads: need a multiple, at most {MAX_GROUP} per KV head")
    if check_positions and b > 0:
        require((pos >= 0).all().reshape(1), "quant_ring_attention: positions must be nonnegative")
    mask = None
    if active is not None:
        check_shape("active", active, (b,), {}, torch.bool)
        if active.device != q.device:
            raise ContractError(f"active is on {active.device}, q on {q.device}")
        mask = active.contiguous()
    ring = cache if inplace and as_is else _writable(cache, inplace)
    q, k, v, pos, on = _aligned(q), _aligned(k), _aligned(v), pos.contiguous(), q.device
    o = torch.empty_like(q)
    if b == 0:
        return o, ring
    nbytes = _workspace_bytes(b, h, hkv, dk, w)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=on) if nbytes else None
    with _lib.on_device(on):
        _lib.call(f"vsp_quant_ring_attn_{_SUFFIX[dtype]}", q.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(),
                  ring.k.data_ptr(), ring.v.data_ptr(), ring.k_scale.data_ptr(), ring.v_scale.data_ptr(),
                  ring.pos.data_ptr(), ring.valid.data_ptr(), o.data_ptr(), _lib.ptr(mask), _lib.ptr(workspace), nbytes,
                  b, h, hkv, dk, w, 1.0 / math.sqrt(dk), 1, _lib.stream_of(on))
    return o, ring
