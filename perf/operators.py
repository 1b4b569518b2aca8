"""The column's few-bit serving operators as cases to be timed: the 4-bit ring, the 8-bit norm and product.

A case is a dict of plain values with a ``kind``:

- ``attn``: one new token per row over a ring held in 4 bits, the token quantised into its slot;
- ``cache``: a chunk of tokens quantised into the ring, and the ring's tokens read back in position order;
- ``norm``: the residual's addition and the RMS norm, its output in 8-bit integers with a scale a row;
- ``project``: a sublayer's projections in 8-bit integers with scales for each token and output channel.

``run`` computes them in plain torch where ``own`` is false and through ``vesper.kernels`` where it is
true; ``exact`` restates each in float64 from the definitions.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path
from typing import Any

import torch
from torch import Tensor

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "vesper-preview_amd"))

Case = dict[str, Any]
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}
EPS = 1e-6  # the norm's epsilon
PEAK_FLOOR = 1e-3  # the norm's floor of a row's peak
TINY = 2.0**-120  # a normalised row of smaller magnitude is stored as zeros

own = False


def listed() -> list[Case]:
    return [
        # one conversation's decode step: the smallest call, all latency
        {"name": "attn_bf16_b1_w512_h8_kv8_d64", "kind": "attn", "dtype": "bf16", "b": 1, "w": 512, "hkv": 8,
         "group": 1, "dk": 64, "fill": 1.0},
        # a batch of 64 conversations, windows full: the decode benchmark's shape
        {"name": "attn_bf16_b64_w512_h8_kv8_d64", "kind": "attn", "dtype": "bf16", "b": 64, "w": 512, "hkv": 8,
         "group": 1, "dk": 64, "fill": 1.0},
        # long windows of an odd size, some not yet full, three query heads a key head, float16
        {"name": "attn_f16_b16_w8191_h12_kv4_d64", "kind": "attn", "dtype": "f16", "b": 16, "w": 8191, "hkv": 4,
         "group": 3, "dk": 64, "fill": 0.6},
        # whole documents in the window, wide heads: the largest cache
        {"name": "attn_bf16_b8_w65536_h16_kv4_d128", "kind": "attn", "dtype": "bf16", "b": 8, "w": 65536, "hkv": 4,
         "group": 4, "dk": 128, "fill": 1.0},
        # one prompt of the window's length into a new ring, read back for its next chunk
        {"name": "cache_bf16_b1_n512_w512_kv8_d64", "kind": "cache", "dtype": "bf16", "b": 1, "n": 512, "w": 512,
         "hkv": 8, "dk": 64, "ragged": False},
        # a padded batch of prompts of different lengths, longer than their ring
        {"name": "cache_bf16_b7_n4097_w4001_kv8_d64", "kind": "cache", "dtype": "bf16", "b": 7, "n": 4097, "w": 4001,
         "hkv": 8, "dk": 64, "ragged": True},
        # a decode step's hidden states
        {"name": "norm_fp32_m64_d512", "kind": "norm", "dtype": "fp32", "rdtype": "bf16", "m": 64, "d": 512, "gain": False},
        # a prefill batch's hidden states at a width of 768, an odd number of tokens
        {"name": "norm_fp32_m32767_d768", "kind": "norm", "dtype": "fp32", "rdtype": "bf16", "m": 32767, "d": 768,
         "gain": True},
        # a decode step's recurrent projections, the write strength among them
        {"name": "project_bf16_m64_d512_rec", "kind": "project", "dtype": "bf16", "m": 64, "d": 512, "h": 8, "hkv": 8,
         "block": "rec"},
        # a few conversations' attention projections of a wide model: bound by the weights
        {"name": "project_f16_m5_d4096_attn", "kind": "project", "dtype": "f16", "m": 5, "d": 4096, "h": 64, "hkv": 16,
         "block": "attn"},
        # a prefill batch's recurrent projections at twelve heads of 64
        {"name": "project_bf16_m32767_d768_rec", "kind": "project", "dtype": "bf16", "m": 32767, "d": 768, "h": 12,
         "hkv": 12, "block": "rec"},
        # the largest product: one square weight over a long prompt
        {"name": "project_bf16_m8192_d8192_one", "kind": "project", "dtype": "bf16", "m": 8192, "d": 8192, "h": 128,
         "hkv": 128, "block": "one"},
    ]


def _spread(rng: random.Random, lo: int, hi: int) -> int:
    """A whole number of ``lo..hi``, even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random) -> Case:
    kind = rng.choices(["attn", "cache", "norm", "project"], [4, 2, 2, 3])[0]
    t = rng.choice(["bf16", "bf16", "f16"])
    if kind == "attn":
        while True:
            c = {"kind": kind, "dtype": t, "b": _spread(rng, 1, 64), "w": _spread(rng, 1, 65536),
                 "hkv": rng.choice([1, 2, 4, 8]), "group": rng.choice([1, 2, 3, 4, 8]),
                 "dk": rng.choice([16, 32, 64, 64, 96, 128, 256]), "fill": round(rng.uniform(0.05, 1.0), 2)}
            if c["b"] * c["w"] * c["hkv"] * c["dk"] <= 1 << 28:
                return c
    if kind == "cache":
        while True:
            c = {"kind": kind, "dtype": t, "b": _spread(rng, 1, 16), "n": _spread(rng, 1, 8192),
                 "w": _spread(rng, 64, 8192), "hkv": rng.choice([1, 2, 4, 8]),
                 "dk": rng.choice([16, 32, 64, 64, 96, 128, 256]), "ragged": rng.random() < 0.5}
            if c["b"] * max(c["n"], c["w"]) * c["hkv"] * c["dk"] <= 14 << 20:
                return c
    if kind == "norm":
        while True:
            x = rng.choice(["fp32", "fp32", "bf16", "f16"])
            c = {"kind": kind, "dtype": x, "rdtype": rng.choice(["bf16", "f16"]) if x == "fp32" else x,
                 "m": _spread(rng, 1, 32768), "d": 8 * _spread(rng, 2, 1024), "gain": rng.random() < 0.5}
            if c["m"] * c["d"] <= 24 << 20:
                return c
    while True:
        h = _spread(rng, 2, 128)
        c = {"kind": kind, "dtype": rng.choice([t, "fp32"]), "m": _spread(rng, 1, 32768),
             "d": 16 * _spread(rng, 8, 512), "h": h, "hkv": rng.choice([k for k in (1, 2, 4, 8, 16) if h % k == 0]),
             "block": rng.choice(["rec", "attn", "one"])}
        n = sum(_used(c))
        if c["m"] * c["d"] * n <= 1 << 39 and c["m"] * n <= 1 << 27:
            return c


def _used(c: Case) -> tuple[int, ...]:
    """The columns of each block of a sublayer's projections, in heads of 64."""
    h, kv = c["h"] * 64, c["hkv"] * 64
    return {"rec": (h, h, h, c["h"]), "attn": (h, kv, kv), "one": (h,)}[c["block"]]


# ---- the 4-bit rows in plain torch --------------------------------------------------------------


def _quantize(x: Tensor) -> tuple[Tensor, Tensor]:
    """Rows ``x [..., dk]`` as codes 0..15 (float32) and the pair ``[..., 2]`` of scale and minimum in x's dtype.

    Each operation is one float32 rounding; the halves keep the largest differences finite."""
    f = x.float() * 0.5
    lo, hi = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    step = ((hi - lo) / torch.full_like(hi, 15.0) * 2.0).to(x.dtype)
    half = step.float() * 0.5
    codes = torch.where(half > 0, torch.round((f - lo) / half).clamp(0, 15), torch.zeros_like(f))
    pair = torch.cat([step, (lo * 2.0).to(x.dtype)], -1)
    fine = torch.isfinite(x).all(-1, keepdim=True)
    return torch.where(fine, codes, torch.zeros_like(codes)), torch.where(fine, pair, torch.full_like(pair, math.nan))


def _pack(codes: Tensor) -> Tensor:
    """Codes ``[..., dk]`` two a byte, the even feature in the low half."""
    c = codes.to(torch.uint8).unflatten(-1, (-1, 2))
    return c[..., 0] | (c[..., 1] << 4)


def _packed(x: Tensor) -> tuple[Tensor, Tensor]:
    codes, pair = _quantize(x)
    return _pack(codes), pair


def _values(packed: Tensor, pair: Tensor) -> Tensor:
    """The float32 values of packed rows and their pairs."""
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).float()
    p = pair.float()
    return p[..., 1:] + p[..., :1] * codes


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g: torch.Generator, *shape: int) -> Tensor:
    return torch.randn(*shape, generator=g, device="cuda")


def _rows(g: torch.Generator, c: Case, n: int) -> Tensor:
    """Keys or values ``[b, n, hkv, dk]``: N(0, 1) about an offset of each channel."""
    return (_randn(g, c["b"], n, c["hkv"], c["dk"]) + 0.5 * _randn(g, 1, 1, c["hkv"], c["dk"])).to(DTYPES[c["dtype"]])


def prepare(case: Case, seed: int) -> dict[str, Any]:
    c, g = case, _gen(seed)
    t = DTYPES[c["dtype"]]
    if c["kind"] == "attn":
        b, w, h = c["b"], c["w"], c["hkv"] * c["group"]
        # rows at positions of their own, from a ring filled in part to one written several times over
        seen = torch.randint(max(1, int(c["fill"] * w)), 3 * w + 1 if c["fill"] < 1 else w + 1, (b, 1), generator=g, device="cuda")
        slot = torch.arange(w, device="cuda").expand(b, w)
        pos = seen - 1 - (seen - 1 - slot) % w
        valid = pos >= 0
        s: dict[str, Any] = {"case": c, "ring_pos": torch.where(valid, pos, torch.zeros_like(pos)), "ring_valid": valid, "pos": seen}
        for name in ("k", "v"):
            codes, pair = _quantize(_rows(g, c, w).transpose(1, 2).contiguous())
            at = valid[:, None, :, None]
            s[f"ring_{name}"] = torch.where(at, _pack(codes), torch.zeros((), dtype=torch.uint8, device="cuda"))
            s[f"ring_{name}_scale"] = torch.where(at, pair, torch.zeros((), dtype=t, device="cuda"))
            s[name] = _rows(g, c, 1)
        s["q"] = _randn(g, b, 1, h, c["dk"]).to(t)
        return s
    if c["kind"] == "cache":
        b, n, w = c["b"], c["n"], c["w"]
        lengths = torch.randint(max(1, n // 2), n + 1, (b,), generator=g, device="cuda") if c["ragged"] else None
        start = torch.randint(0, 2 * w, (b, 1), generator=g, device="cuda")
        last = start + (n if lengths is None else lengths[:, None])
        asked = last - w + torch.arange(w, device="cuda")  # the window's positions in order, oldest first
        zeros = [torch.zeros(b, c["hkv"], w, c["dk"] // 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
        pairs = [torch.zeros(b, c["hkv"], w, 2, dtype=t, device="cuda") for _ in range(2)]
        return {"case": c, "k": _rows(g, c, n), "v": _rows(g, c, n), "pos": start + torch.arange(n, device="cuda"),
                "lengths": lengths, "asked": asked, "ring_k": zeros[0], "ring_v": zeros[1], "ring_k_scale": pairs[0],
                "ring_v_scale": pairs[1], "ring_pos": torch.zeros(b, w, dtype=torch.long, device="cuda"),
                "ring_valid": torch.zeros(b, w, dtype=torch.bool, device="cuda")}
    if c["kind"] == "norm":
        m, d = c["m"], c["d"]
        # a residual stream: rows of different magnitude, a few channels larger than the others
        x = _randn(g, m, d) * torch.exp(_randn(g, m, 1)) * torch.exp(0.7 * _randn(g, 1, d))
        return {"case": c, "x": x.to(t), "residual": _randn(g, m, d).to(DTYPES[c["rdtype"]]),
                "gain": torch.exp(0.2 * _randn(g, d)) if c["gain"] else None}
    used = _used(c)
    m, d, cols = c["m"], c["d"], max(used)
    z = torch.randint(-127, 128, (m, d), generator=g, device="cuda", dtype=torch.int8)
    weights = torch.randint(-127, 128, (len(used), cols, d), generator=g, device="cuda", dtype=torch.int8)
    # scales of N(0, 1) rows and N(0, 1 / d) weights, whose largest element is about 3.5 deviations
    return {"case": c, "z": z, "z_scale": 3.5 / 127 * torch.exp(0.2 * _randn(g, m)), "weights": weights,
            "weights_scale": 3.5 / 127 / math.sqrt(d) * torch.exp(0.2 * _randn(g, len(used), cols)), "used": used}


def run(state: dict[str, Any]) -> Any:
    s, c = state, state["case"]
    if c["kind"] == "attn":
        return _attn_own(s, c) if own else _attn(s, c)
    if c["kind"] == "cache":
        return _cache_own(s, c) if own else _cache(s, c)
    if c["kind"] == "norm":
        return _norm_own(s, c) if own else _norm(s, c)
    return _project_own(s, c) if own else _project(s, c)


# ---- the framework's calls ----------------------------------------------------------------------


def _ring(s: dict[str, Any], c: Case) -> Any:
    from vesper.kernels.ring_quant import QuantRingKVCache

    return QuantRingKVCache(s["ring_k"], s["ring_v"], s["ring_k_scale"], s["ring_v_scale"], s["ring_pos"],
                            s["ring_valid"], c["w"])


def _attn_own(s: dict[str, Any], c: Case) -> Any:
    from vesper.kernels.ring_quant import quant_ring_attention

    o, ring = quant_ring_attention(s["q"], s["k"], s["v"], s["pos"], _ring(s, c), inplace=True, check_positions=False)
    return [o, ring.k, ring.v, ring.k_scale, ring.v_scale, ring.pos, ring.valid]


def _cache_own(s: dict[str, Any], c: Case) -> Any:
    from vesper.kernels.ring_quant import quant_ring_read, quant_ring_write

    ring = quant_ring_write(s["k"], s["v"], s["pos"], _ring(s, c), lengths=s["lengths"], inplace=True, check_positions=False)
    keys, values, found = quant_ring_read(ring, s["asked"])
    return [keys, values, found, ring.pos, ring.valid]


def _norm_own(s: dict[str, Any], c: Case) -> Any:
    from vesper.kernels.norm import rms_norm_int8

    total = torch.empty_like(s["x"])
    codes, scale = rms_norm_int8(s["x"], s["gain"], residual=s["residual"], sum_out=total)
    # the codes as the values they stand for
    values = torch.empty(codes.shape, dtype=torch.bfloat16, device=codes.device)
    return [torch.mul(codes, scale.unsqueeze(-1), out=values), scale, total]


def _project_own(s: dict[str, Any], c: Case) -> Any:
    from vesper.kernels.norm import projection_int8

    return projection_int8(s["z"], s["z_scale"], s["weights"], s["weights_scale"], s["used"],
                           sigmoid_block=3 if c["block"] == "rec" else None, dtype=DTYPES[c["dtype"]])


# ---- the plain forms ----------------------------------------------------------------------------


def _store(s: dict[str, Any], rows: Tensor, at: Tensor, pos: Tensor, k: Tensor, v: Tensor) -> None:
    """Tokens ``k``, ``v`` at positions ``pos`` quantised into slots ``at`` of the batch rows ``rows``."""
    s["ring_k"][rows, :, at], s["ring_k_scale"][rows, :, at] = _packed(k)
    s["ring_v"][rows, :, at], s["ring_v_scale"][rows, :, at] = _packed(v)
    s["ring_pos"][rows, at] = pos
    s["ring_valid"][rows, at] = True


def _attn(s: dict[str, Any], c: Case) -> Any:
    """Scores over the ring's values, a softmax with the new token, its weighted values; then the write."""
    b, w, hkv, dk, group = c["b"], c["w"], c["hkv"], c["dk"], c["group"]
    p = s["pos"]
    slot = torch.arange(w, device=p.device)
    seen = s["ring_valid"] & (s["ring_pos"] <= p) & (s["ring_pos"] > p - w) & (slot != p % w)
    keys = _values(s["ring_k"], s["ring_k_scale"])  # [b, hkv, w, dk]
    values = _values(s["ring_v"], s["ring_v_scale"])
    q = s["q"].float().view(b, hkv, group, dk)
    scores = torch.matmul(q, keys.transpose(2, 3).contiguous()) / math.sqrt(dk)
    scores = scores.masked_fill(~seen[:, None, None, :], -math.inf)
    new = (q * s["k"].float().transpose(1, 2)).sum(-1, keepdim=True) / math.sqrt(dk)
    top = torch.maximum(scores.amax(-1, keepdim=True), new)
    weights, mine = torch.exp(scores - top), torch.exp(new - top)
    total = weights.sum(-1, keepdim=True) + mine
    o = (torch.matmul(weights, values) + mine * s["v"].float().transpose(1, 2)) / total
    _store(s, torch.arange(b, device=p.device), (p % w)[:, 0], p[:, 0], s["k"][:, 0], s["v"][:, 0])
    return [o.view(b, 1, hkv * group, dk).to(s["q"].dtype), s["ring_k"], s["ring_v"], s["ring_k_scale"],
            s["ring_v_scale"], s["ring_pos"], s["ring_valid"]]


def _written(s: dict[str, Any], c: Case) -> tuple[Tensor, Tensor]:
    """The batch rows and the tokens that the ring keeps of the chunk: each row's last ``w`` of its length."""
    n, w = c["n"], c["w"]
    i = torch.arange(n, device=s["k"].device).expand(c["b"], n)
    length = torch.full((c["b"], 1), n, device=i.device) if s["lengths"] is None else s["lengths"][:, None]
    return torch.nonzero((i < length) & (i >= length - w), as_tuple=True)


def _cache(s: dict[str, Any], c: Case) -> Any:
    t, w = DTYPES[c["dtype"]], c["w"]
    rows, token = _written(s, c)
    pos = s["pos"][rows, token]
    _store(s, rows, pos % w, pos, s["k"][rows, token], s["v"][rows, token])
    slot = s["asked"] % w
    row = torch.arange(c["b"], device=slot.device)[:, None]
    found = s["ring_valid"][row, slot] & (s["ring_pos"][row, slot] == s["asked"])
    top = torch.finfo(t).max
    keys, values = ((_values(s[f"ring_{name}"][row, :, slot], s[f"ring_{name}_scale"][row, :, slot]).clamp(-top, top)
                     * found[:, :, None, None]).to(t) for name in ("k", "v"))
    return [keys, values, found, s["ring_pos"], s["ring_valid"]]


def _norm(s: dict[str, Any], c: Case) -> Any:
    total = s["x"].float() + s["residual"].float()
    peak = total.abs().amax(-1, keepdim=True).clamp_min(PEAK_FLOOR)
    u = total / peak
    y = u / torch.sqrt(u.square().mean(-1, keepdim=True) + EPS / peak.square())
    if s["gain"] is not None:
        y = y * s["gain"]
    top = y.abs().amax(-1, keepdim=True)
    scale = torch.where(top < TINY, torch.zeros_like(top), top / torch.full_like(top, 127.0))
    codes = torch.where(scale > 0, torch.round(y / scale), torch.zeros_like(y))
    return [(codes * scale).bfloat16(), scale[:, 0], total.to(s["x"].dtype)]


def _project(s: dict[str, Any], c: Case) -> Any:
    z = s["z"].float()
    outs = [torch.matmul(z, s["weights"][j, :u].float().t()) * (s["z_scale"][:, None] * s["weights_scale"][j, :u])
            for j, u in enumerate(s["used"])]
    return [(torch.sigmoid(y) if c["block"] == "rec" and j == 3 else y).to(DTYPES[c["dtype"]]) for j, y in enumerate(outs)]


# ---- from the definitions, in float64 -----------------------------------------------------------


def work(case: Case) -> dict[str, float]:
    c = case
    size = torch.finfo(DTYPES[c["dtype"]]).bits // 8
    if c["kind"] == "attn":
        b, w, hkv, dk = c["b"], c["w"], c["hkv"], c["dk"]
        filled = w if c["fill"] >= 1 else w * (1 - (1 - c["fill"]) ** 2 / (2 * (3 - c["fill"])))
        ring = b * filled * hkv * (dk + 8) + b * w * 9  # codes and pairs of keys and values; positions and flags
        return {"bytes": ring + 2 * b * hkv * c["group"] * dk * 2 + b * hkv * dk * 5,
                "flops": 4.0 * b * filled * hkv * c["group"] * dk}
    if c["kind"] == "cache":
        kept = c["b"] * min(c["w"], c["n"] * (0.75 if c["ragged"] else 1.0)) * c["hkv"]
        rows = c["b"] * c["w"]
        # rows in, codes and pairs out; then the codes and pairs in, the whole window out
        return {"bytes": kept * (4 * c["dk"] + 2 * (c["dk"] + 8)) + rows * (4 * c["hkv"] * c["dk"] + 27), "flops": kept * 20.0 * c["dk"]}
    if c["kind"] == "norm":
        rbits = torch.finfo(DTYPES[c["rdtype"]]).bits // 8
        return {"bytes": c["m"] * c["d"] * (2 * size + rbits + 1 + 2) + 4 * c["m"], "flops": 10.0 * c["m"] * c["d"]}
    n = sum(_used(c))
    return {"bytes": c["m"] * c["d"] + n * c["d"] + c["m"] * n * size + 4 * (c["m"] + n), "flops": 2.0 * c["m"] * c["d"] * n}


def exact(case: Case, seed: int) -> Any:
    s, c = prepare(case, seed), case
    if c["kind"] == "attn":
        if c["b"] * c["w"] * c["hkv"] * c["dk"] > 1 << 28:
            return None
        return _exact_attn(s, c)
    if c["kind"] == "cache":
        return _exact_cache(s, c)
    if c["kind"] == "norm":
        total = s["x"].double() + s["residual"].double()
        y = total / torch.sqrt(total.square().mean(-1, keepdim=True) + EPS)
        if s["gain"] is not None:
            y = y * s["gain"].double()
        scale = y.abs().amax(-1, keepdim=True) / 127
        return [torch.round(y / scale.clamp_min(1e-300)) * scale, scale[:, 0], total]
    z = s["z"].double() * s["z_scale"].double()[:, None]
    outs = []
    for j, u in enumerate(s["used"]):
        w = s["weights"][j, :u].double() * s["weights_scale"][j, :u].double()[:, None]
        y = z @ w.t()
        outs.append(1 / (1 + torch.exp(-y)) if c["block"] == "rec" and j == 3 else y)
    return outs


def _exact_attn(s: dict[str, Any], c: Case) -> Any:
    b, w, dk = c["b"], c["w"], c["dk"]
    out = torch.empty(b, 1, c["hkv"] * c["group"], dk, dtype=torch.float64, device="cuda")
    slots = torch.arange(w, device="cuda")
    scales = [s["ring_k_scale"].double(), s["ring_v_scale"].double()]
    for i in range(b):
        p = int(s["pos"][i, 0])
        use = s["ring_valid"][i] & (s["ring_pos"][i] <= p) & (s["ring_pos"][i] > p - w) & (slots != p % w)
        for kv in range(c["hkv"]):
            rows = []
            for name, pair in zip(("k", "v"), scales):
                packed = s[f"ring_{name}"][i, kv, use].long()
                low_high = torch.empty(packed.shape[0], dk, dtype=torch.float64, device="cuda")
                low_high[:, 0::2], low_high[:, 1::2] = (packed % 16).double(), (packed // 16).double()
                x = low_high * pair[i, kv, use, 0:1] + pair[i, kv, use, 1:2]
                rows.append(torch.cat([x, s[name][i, :, kv].double()]))  # and the new token
            heads = slice(kv * c["group"], (kv + 1) * c["group"])
            weights = torch.softmax(s["q"][i, 0, heads].double() @ rows[0].t() / math.sqrt(dk), -1)
            out[i, 0, heads] = weights @ rows[1]
        for name, pair in zip(("k", "v"), scales):
            x = s[name][i, 0].double()
            pair[i, :, p % w, 0] = (x.amax(-1) - x.amin(-1)) / 15
            pair[i, :, p % w, 1] = x.amin(-1)
    return [out, None, None, *scales, None, None]


def _exact_cache(s: dict[str, Any], c: Case) -> Any:
    b, w, t = c["b"], c["w"], DTYPES[c["dtype"]]
    keys, values = (torch.zeros(b, w, c["hkv"], c["dk"], dtype=torch.float64, device="cuda") for _ in range(2))
    for i in range(b):
        n = c["n"] if s["lengths"] is None else int(s["lengths"][i])
        kept = min(n, w)
        for out, name in ((keys, "k"), (values, "v")):
            x = s[name][i, n - kept:n].double()
            lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
            step = ((hi - lo) / 15).to(t).double()  # held in the cache's type
            codes = torch.round((x - lo) / step.clamp_min(1e-300)).clamp(0, 15)
            out[i, w - kept:] = lo + step * codes
    return [keys, values, None, None, None]
