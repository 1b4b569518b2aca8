"""The gated recurrence's operators as cases to be timed: the gated delta rule's scan, its step, and the layer norm.

A case is a dict of plain values with a ``kind``:

- ``step``: one token a row through the gated delta rule, the state updated in place (decoding);
- ``scan``: the gated delta rule over a block of tokens from a given state (prefill);
- ``train``: the scan and its backward pass: outputs, the state after the block, and every input's gradient;
- ``norm``: the residual's addition and the layer norm, the sum kept for the next sublayer;
- ``norm_train``: that and its backward pass, the weight's and the bias's gradients among the outputs.

``run`` computes them in plain torch where ``own`` is false and through ``vesper.kernels`` where it is
true; ``exact`` restates each in float64 from the definitions, the scan token by token.
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
EPS = 1e-5  # the layer norm's epsilon
CHUNK = 64  # tokens of a chunk of the plain scan
LEAST = -1e4  # log decays below it count as it: exp is zero either way

own = False


def listed() -> list[Case]:
    return [
        # one conversation's decode step: the smallest call, all latency
        {"name": "step_bf16_b1_h8_d64", "kind": "step", "dtype": "bf16", "b": 1, "h": 8, "dk": 64},
        # a batch of 64 conversations: the decode benchmark's shape
        {"name": "step_bf16_b64_h8_d64", "kind": "step", "dtype": "bf16", "b": 64, "h": 8, "dk": 64},
        # many conversations of a model with wide heads in float32: bound by the states
        {"name": "step_fp32_b200_h16_d128", "kind": "step", "dtype": "fp32", "b": 200, "h": 16, "dk": 128},
        # a prompt's last piece carried on from a state, float32: the parity configuration
        {"name": "scan_fp32_b2_n512_h4_d64", "kind": "scan", "dtype": "fp32", "b": 2, "n": 512, "h": 4, "dk": 64, "resets": False},
        # the prefill benchmark's shape
        {"name": "scan_bf16_b8_n4096_h8_d64", "kind": "scan", "dtype": "bf16", "b": 8, "n": 4096, "h": 8, "dk": 64, "resets": False},
        # one long document of an odd length, twelve heads; packed with others (the state forgotten at their starts)
        {"name": "scan_bf16_b1_n8191_h12_d64", "kind": "scan", "dtype": "bf16", "b": 1, "n": 8191, "h": 12, "dk": 64, "resets": True},
        # a training batch: the configuration's chunk, heads and width
        {"name": "train_bf16_b16_n1024_h12_d64", "kind": "train", "dtype": "bf16", "b": 16, "n": 1024, "h": 12, "dk": 64, "resets": False},
        # short float32 sequences of narrow heads
        {"name": "train_fp32_b32_n88_h2_d16", "kind": "train", "dtype": "fp32", "b": 32, "n": 88, "h": 2, "dk": 16, "resets": False},
        # wide heads, an odd length, packed documents
        {"name": "train_bf16_b2_n1500_h8_d128", "kind": "train", "dtype": "bf16", "b": 2, "n": 1500, "h": 8, "dk": 128, "resets": True},
        # a decode step's hidden states
        {"name": "norm_fp32_m64_d512", "kind": "norm", "dtype": "fp32", "rdtype": "bf16", "ydtype": "bf16", "m": 64, "d": 512},
        # a training batch's hidden states at a width of 768, an odd number of tokens
        {"name": "norm_train_fp32_m16383_d768", "kind": "norm_train", "dtype": "fp32", "rdtype": "bf16", "ydtype": "bf16",
         "m": 16383, "d": 768},
        # the largest: bfloat16 throughout, a wide model's
        {"name": "norm_train_bf16_m16384_d4096", "kind": "norm_train", "dtype": "bf16", "rdtype": "bf16", "ydtype": "bf16",
         "m": 16384, "d": 4096},
    ]


def _spread(rng: random.Random, lo: int, hi: int) -> int:
    """A whole number of ``lo..hi``, even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random) -> Case:
    kind = rng.choices(["step", "scan", "train", "norm", "norm_train"], [2, 3, 3, 1, 2])[0]
    if kind in ("norm", "norm_train"):
        while True:
            x = rng.choice(["fp32", "fp32", "bf16", "f16"])
            c = {"kind": kind, "dtype": x, "rdtype": rng.choice(["bf16", "f16", "fp32"]) if x == "fp32" else x,
                 "ydtype": rng.choice(["bf16", "f16", "fp32"]) if x == "fp32" else x,
                 "m": _spread(rng, 1, 65536), "d": rng.choice([1, 8, 8, 8]) * _spread(rng, 2, 1024)}
            if c["m"] * c["d"] <= 32 << 20:
                return c
    t = rng.choice(["bf16", "bf16", "fp32"])
    widths = [8, 16, 32, 40, 64, 64, 96, 128, 128, 256]
    if kind == "step":
        while True:
            c = {"kind": kind, "dtype": t, "b": _spread(rng, 1, 512), "h": _spread(rng, 1, 32), "dk": rng.choice(widths)}
            if c["b"] * c["h"] * c["dk"] ** 2 <= 200 * 16 * 128 ** 2:
                return c
    while True:
        c = {"kind": kind, "dtype": t, "b": _spread(rng, 1, 64), "n": _spread(rng, 1, 8192), "h": _spread(rng, 1, 16),
             "dk": rng.choice(widths), "resets": rng.random() < 0.4}
        elements = c["b"] * c["n"] * c["h"] * c["dk"]
        # the wide heads' work grows with their width, the float32 products' with the type
        cost = elements * max(1.0, c["dk"] / 64) * (2 if t == "fp32" else 1)
        if cost <= (12 << 20 if kind == "train" else 16 << 20) and c["b"] * c["h"] * c["dk"] ** 2 <= 1 << 24:
            return c


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g: torch.Generator, *shape: int) -> Tensor:
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case: Case, seed: int) -> dict[str, Any]:
    c, gen = case, _gen(seed)
    t = DTYPES[c["dtype"]]
    if c["kind"] in ("norm", "norm_train"):
        m, d = c["m"], c["d"]
        # a residual stream: rows of different magnitude about a mean of their own, a few channels larger than the others
        x = _randn(gen, m, d) * torch.exp(0.7 * _randn(gen, 1, d)) * torch.exp(_randn(gen, m, 1)) + _randn(gen, m, 1)
        s = {"case": c, "x": x.to(t), "residual": _randn(gen, m, d).to(DTYPES[c["rdtype"]]),
             "gain": torch.exp(0.2 * _randn(gen, d)), "bias": 0.1 * _randn(gen, d)}
        if c["kind"] == "norm_train":
            s["dy"] = _randn(gen, m, d).to(DTYPES[c["ydtype"]])
            s["dsum"] = (0.3 * _randn(gen, m, d)).to(t)
            for name in ("x", "residual", "gain", "bias"):
                s[name].requires_grad_()
        return s
    b, h, dk = c["b"], c["h"], c["dk"]
    lead = (b, h) if c["kind"] == "step" else (b, c["n"], h)
    k = _randn(gen, *lead, dk) + 0.3 * _randn(gen, h, dk)
    k = k / k.norm(dim=-1, keepdim=True).clamp_min(1.0)
    # log decays of a softplus gate, a rate a head: some remember thousands of tokens, some a few
    rate = torch.exp(torch.empty(h, device="cuda").uniform_(math.log(1e-3), math.log(2.0), generator=gen))
    g = -rate * torch.nn.functional.softplus(_randn(gen, *lead))
    if c.get("resets"):  # documents of about 200 tokens, packed: the state forgotten before a document's first token
        start = torch.rand(b, c["n"], 1, generator=gen, device="cuda") < 1 / 200
        g = g.masked_fill(start, -math.inf)
    s = {"case": c, "q": _randn(gen, *lead, dk).to(t), "k": k.to(t), "v": _randn(gen, *lead, dk).to(t),
         "beta": torch.sigmoid(_randn(gen, *lead)).to(t), "g": g, "state": 0.5 * _randn(gen, b, h, dk, dk)}
    if c["kind"] == "train":
        s["do"] = _randn(gen, *lead, dk).to(t)
        s["dstate"] = 0.3 * _randn(gen, b, h, dk, dk)
        for name in LEAVES:
            s[name].requires_grad_()
    return s


LEAVES = ("q", "k", "v", "beta", "g", "state")


def run(state: dict[str, Any]) -> Any:
    s, c = state, state["case"]
    if c["kind"] == "step":
        return _step_own(s) if own else _step(s)
    if c["kind"] == "scan":
        return _scan_own(s) if own else _scan(*(s[name] for name in LEAVES))
    if c["kind"] == "train":
        o, after = _scan_own(s) if own else _scan(*(s[name] for name in LEAVES))
        return [o, after, *torch.autograd.grad([o, after], [s[name] for name in LEAVES], [s["do"], s["dstate"]])]
    y, total = _norm_own(s, c) if own else _norm(s, c)
    if c["kind"] == "norm":
        return [y, total]
    return [y, total, *torch.autograd.grad([y, total], [s["x"], s["residual"], s["gain"], s["bias"]], [s["dy"], s["dsum"]])]


# ---- the framework's calls ----------------------------------------------------------------------


def _step_own(s: dict[str, Any]) -> Any:
    from vesper.kernels.gated_scan import gated_delta_step

    return list(gated_delta_step(s["q"], s["k"], s["v"], s["beta"], s["g"], s["state"], out_state=s["state"]))


def _scan_own(s: dict[str, Any]) -> Any:
    from vesper.kernels.gated_scan import gated_delta_scan

    return list(gated_delta_scan(s["q"], s["k"], s["v"], s["beta"], s["g"], s["state"]))


def _norm_own(s: dict[str, Any], c: Case) -> Any:
    from vesper.kernels.layer_norm import layer_norm

    return layer_norm(s["x"], s["gain"], s["bias"], residual=s["residual"], eps=EPS, dtype=DTYPES[c["ydtype"]])


# ---- the plain forms ----------------------------------------------------------------------------


def _step(s: dict[str, Any]) -> Any:
    """The decayed state reads the key, takes the correction, and reads the query."""
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    kept = torch.exp(s["g"])[..., None, None] * s["state"]
    u = s["beta"].float()[..., None] * (v - (kept * k[..., None]).sum(-2))
    s["state"].copy_(kept + k[..., None] * u[..., None, :])
    return [(s["state"] * q[..., None]).sum(-2).to(s["q"].dtype), s["state"]]


def _inverse(a: Tensor) -> Tensor:
    """``(I + a)^-1`` of strictly lower triangles ``[..., C, C]``: inverses of diagonal blocks, joined two by two."""
    c = a.shape[-1]
    x = torch.ones(*a.shape[:-2], c, 1, 1, dtype=a.dtype, device=a.device)  # [..., blocks, size, size]
    size = 1
    while size < c:
        low = a.unflatten(-2, (c // size, size)).unflatten(-1, (c // size, size)).movedim(-2, -3)
        block = torch.arange(0, c // size, 2, device=a.device)
        first, second = x[..., block, :, :], x[..., block + 1, :, :]
        corner = -(second @ low[..., block + 1, block, :, :] @ first)
        x = torch.cat([torch.cat([first, torch.zeros_like(first)], -1), torch.cat([corner, second], -1)], -2)
        size *= 2
    return x[..., 0, :, :]


def _scan(q: Tensor, k: Tensor, v: Tensor, beta: Tensor, g: Tensor, state: Tensor) -> list[Tensor]:
    """Chunks of ``CHUNK`` tokens: within them by products of all pairs of tokens, from one to the next by the state."""
    b, n, h, dk = q.shape
    chunks = -(-n // CHUNK)

    def split(x: Tensor) -> Tensor:  # [b, h, chunks, CHUNK, ...], zeros behind the last token
        x = torch.cat([x, x.new_zeros(b, chunks * CHUNK - n, *x.shape[2:])], 1)
        return x.unflatten(1, (chunks, CHUNK)).movedim(3, 1)

    qc, kc, vc, bc = (split(x.float()) for x in (q, k, v, beta))
    # sums of logarithms and their differences in float64: a decayed-away token's sum is large, its neighbours' differences are not
    total = torch.cumsum(split(g.double().clamp_min(LEAST)), -1)
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    pair = (total[..., :, None] - total[..., None, :]).masked_fill(~lower, -math.inf)
    decay = torch.exp(pair.float())  # [.., i, j]: what is left at token i of what token j wrote
    since, until, whole = (torch.exp(x.float())[..., None] for x in (total, total[..., -1:] - total, total[..., -1:]))
    keys_t = kc.transpose(-1, -2).contiguous()
    solved = _inverse(torch.tril(bc[..., None] * decay * (kc @ keys_t), -1))
    reads = decay * (qc @ keys_t)
    bv, bk = bc[..., None] * vc, bc[..., None] * since * kc
    kept, queries = until * kc, since * qc
    outs = []
    for i in range(chunks):
        delta = solved[:, :, i] @ (bv[:, :, i] - bk[:, :, i] @ state)
        outs.append(queries[:, :, i] @ state + reads[:, :, i] @ delta)
        state = whole[:, :, i] * state + kept[:, :, i].transpose(-1, -2) @ delta
    o = torch.stack(outs, 2).movedim(1, 3).flatten(1, 2)[:, :n]
    return [o.to(q.dtype), state]


def _norm(s: dict[str, Any], c: Case) -> Any:
    total = s["x"].float() + s["residual"].float()
    centred = total - total.mean(-1, keepdim=True)
    y = centred / torch.sqrt(centred.square().mean(-1, keepdim=True) + EPS) * s["gain"] + s["bias"]
    return [y.to(DTYPES[c["ydtype"]]), total.to(s["x"].dtype)]


# ---- from the definitions, in float64 -----------------------------------------------------------


def work(case: Case) -> dict[str, float]:
    c = case
    size = torch.finfo(DTYPES[c["dtype"]]).bits // 8
    if c["kind"] in ("norm", "norm_train"):
        r, y = (torch.finfo(DTYPES[c[name]]).bits // 8 for name in ("rdtype", "ydtype"))
        forward, backward = 2 * size + r + y, 2 * size + y + r  # x, r in, the sum and y out; dy, dsum in, dx, dr out
        train = c["kind"] == "norm_train"
        return {"bytes": c["m"] * c["d"] * (forward + (backward if train else 0)) + (16 if train else 8) * c["d"],
                "flops": (25.0 if train else 9.0) * c["m"] * c["d"]}
    b, h, dk = c["b"], c["h"], c["dk"]
    tokens, states = b * c.get("n", 1) * h, b * h * dk * dk
    forward = tokens * (4 * dk * size + size + 4) + 8 * states
    if c["kind"] != "train":
        return {"bytes": forward, "flops": 7.0 * tokens * dk * dk}
    # back: do in, five gradients out, the state's gradient in and out (q, k, v, beta and g are read once for both)
    return {"bytes": forward + tokens * (4 * dk * size + size + 4) + 8 * states, "flops": 21.0 * tokens * dk * dk}


def exact(case: Case, seed: int) -> Any:
    s, c = prepare(case, seed), case
    with torch.no_grad():
        if c["kind"] in ("norm", "norm_train"):
            return _exact_norm(s, c)
        if c["kind"] == "step":
            o, state = _exact_token(*(s[name].double() for name in LEAVES))[:2]
            return [o, state]
        if c["kind"] == "train" and c["b"] * c["n"] * c["h"] * c["dk"] ** 2 > 1 << 31:
            return None
        return _exact_scan(s, c)


def _exact_token(q: Tensor, k: Tensor, v: Tensor, beta: Tensor, g: Tensor, state: Tensor) -> tuple[Tensor, ...]:
    faded = g.exp()[..., None, None] * state
    error = v - (k[..., None, :] @ faded)[..., 0, :]
    after = faded + beta[..., None, None] * k[..., :, None] * error[..., None, :]
    return (q[..., None, :] @ after)[..., 0, :], after, faded, error


def _exact_scan(s: dict[str, Any], c: Case) -> Any:
    q, k, v, beta, g, state = (s[name].double() for name in LEAVES)
    train, tokens = c["kind"] == "train", range(c["n"])
    outs, before = [], []
    for t in tokens:
        if train:
            before.append(state)
        o, state = _exact_token(q[:, t], k[:, t], v[:, t], beta[:, t], g[:, t], state)[:2]
        outs.append(o)
    if not train:
        return [torch.stack(outs, 1), state]
    do, ds = s["do"].double(), s["dstate"].double()
    dq, dk, dv, db, dg = (torch.empty_like(x) for x in (q, k, v, beta, g))
    for t in reversed(tokens):
        kt, bt = k[:, t], beta[:, t]
        _, after, faded, error = _exact_token(q[:, t], kt, v[:, t], bt, g[:, t], before[t])
        ds = ds + q[:, t][..., :, None] * do[:, t][..., None, :]
        dq[:, t] = (after @ do[:, t][..., :, None])[..., 0]
        wrote = (kt[..., None, :] @ ds)[..., 0, :]  # the gradient of beta * error
        db[:, t] = (wrote * error).sum(-1)
        dv[:, t] = bt[..., None] * wrote
        dk[:, t] = bt[..., None] * ((ds @ error[..., :, None]) - (faded @ wrote[..., :, None]))[..., 0]
        dfaded = ds - bt[..., None, None] * kt[..., :, None] * wrote[..., None, :]
        dg[:, t] = (dfaded * faded).sum((-1, -2))
        ds = g[:, t].exp()[..., None, None] * dfaded
    return [torch.stack(outs, 1), state, dq, dk, dv, db, dg, ds]


def _exact_norm(s: dict[str, Any], c: Case) -> Any:
    total = s["x"].double() + s["residual"].double()
    var, mean = torch.var_mean(total, -1, correction=0, keepdim=True)
    root = (var + EPS).rsqrt()
    unit = root * (total - mean)
    gain = s["gain"].double()
    y = unit * gain + s["bias"].double()
    if c["kind"] == "norm":
        return [y, total]
    # the backward pass starts from the sum as it is kept, in x's type
    dy = s["dy"].double()
    w = dy * gain
    dx = root * (w - w.mean(-1, keepdim=True) - unit * (w * unit).mean(-1, keepdim=True)) + s["dsum"].double()
    return [y, total, dx, dx, (dy * unit).sum(0), dy.sum(0)]
