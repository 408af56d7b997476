"""Operators of an encoder layer that rotates its heads and projects in 8 bits.

Rotary positions of queries and keys (forward and with gradients), token
vectors held as 8-bit integers with a scale each and read back, and the linear
layer on such integers with its epilogues: what a late-interaction model runs
between its norms, its attention and its index when a corpus is encoded, when
one query is, and (the rotation) when the model is trained. ``run`` computes a
case in its plain form (elementary torch operations) or, with ``own`` set,
through ``late_interaction_kernels.encoder``.

``listed`` names eleven cases, ``draw`` gives another of the same ranges,
``prepare`` makes what a program holds before the call, ``run`` is the call,
``exact`` the same outputs in 64-bit floating point.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "int8": torch.int8}
_EB = {"bf16": 2, "fp16": 2, "fp32": 4, "int8": 1}


def listed():
    return [
        # One user query of 32 tokens: q and k of one layer, where the latency
        # of the call counts.
        {"name": "rotary_query", "kind": "rotary", "dtype": "bf16", "n": 1, "len": 32, "h": 12, "hk": 12, "d": 64,
         "r": 64, "pos": "count", "far": 0, "inter": False, "base": 10000.0, "factor": 1.0, "train": False},
        # One new token for each of 256 texts at far positions of their own,
        # shared wide heads, frequencies scaled for long contexts.
        {"name": "rotary_single_tokens", "kind": "rotary", "dtype": "fp16", "n": 256, "len": 1, "h": 16, "hk": 4,
         "d": 128, "r": 128, "pos": "given", "far": 131072, "inter": True, "base": 10000.0, "factor": 8.0,
         "train": False},
        # Encoding packed passages and long documents.
        {"name": "rotary_packed", "kind": "rotary", "dtype": "bf16", "n": 256, "len": 300, "h": 12, "hk": 12, "d": 64,
         "r": 64, "pos": "packed", "far": 0, "inter": False, "base": 160000.0, "factor": 1.0, "train": False},
        # Training step on 16 page images of 1030 patches, shared wide heads of
        # which a half is rotated.
        {"name": "rotary_train_pages", "kind": "rotary", "dtype": "bf16", "n": 16, "len": 1030, "h": 16, "hk": 4,
         "d": 128, "r": 64, "pos": "count", "far": 0, "inter": False, "base": 10000.0, "factor": 1.0, "train": True},
        # The tokens of one query, held in 8 bits and read back.
        {"name": "tokens8_query", "kind": "tokens8", "dtype": "bf16", "rows": 32, "d": 768},
        # A shard of an index: a million token vectors of 128.
        {"name": "tokens8_index", "kind": "tokens8", "dtype": "fp16", "rows": 1030001, "d": 128},
        # Hidden states in full precision, rows of an odd length.
        {"name": "tokens8_hidden_fp32", "kind": "tokens8", "dtype": "fp32", "rows": 32961, "d": 1027},
        # One query through the joint projection of q, k and v: the weights are
        # read for 32 rows.
        {"name": "linear8_query", "kind": "linear8", "x": "bf16", "out": "bf16", "rows": 32, "k": 768, "n": 2304,
         "act": "", "gated": False, "bias": True, "residual": False},
        # The joint projection for the valid tokens of 256 passages, encoding.
        {"name": "linear8_passages", "kind": "linear8", "x": "fp16", "out": "fp16", "rows": 44801, "k": 768, "n": 2304,
         "act": "", "gated": False, "bias": True, "residual": False},
        # The way out of the feed-forward block with the residual sum.
        {"name": "linear8_residual", "kind": "linear8", "x": "bf16", "out": "bf16", "rows": 44801, "k": 1152, "n": 768,
         "act": "", "gated": False, "bias": False, "residual": True},
        # The way into a wide gated block on 16 page images, tokens quantised
        # once before.
        {"name": "linear8_gated_pages", "kind": "linear8", "x": "int8", "out": "bf16", "rows": 16480, "k": 1024,
         "n": 2816, "act": "silu", "gated": True, "bias": False, "residual": False},
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n if n < 2048 else n - 1 + n % 2  # long ones are odd: no whole tiles


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "rotary", "tokens8", "tokens8", "linear8", "linear8", "linear8"])
    if kind == "rotary":
        h, hk, d, r = rng.choice([(12, 12, 64, 64), (16, 4, 128, 128), (16, 4, 128, 64), (16, 16, 72, 72),
                                  (6, 6, 32, 32), (8, 8, 96, 24), (12, 4, 64, 32), (14, 2, 80, 20)])
        train = rng.random() < 0.4
        dtype, pos = rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice(["count", "given", "packed"])
        # fewer elements of q and k than the largest listed case has
        tokens = _log(rng, 1, (24 << 20) // ((h + hk) * d) * (1 if train or dtype == "fp32" else 2))
        length = 1 if pos == "given" and not train and rng.random() < 0.4 else _log(rng, 1, min(tokens, 4096))
        return {"kind": kind, "dtype": dtype, "n": max(1, tokens // length), "len": length, "h": h, "hk": hk, "d": d,
                "r": r, "pos": pos, "far": _log(rng, 1, 1 << 20) if pos == "given" else 0,
                "inter": rng.random() < 0.5, "base": rng.choice([10000.0, 160000.0, 1000000.0]),
                "factor": rng.choice([1.0, 1.0, 4.0, 8.0]), "train": train}
    if kind == "tokens8":
        d = rng.choice([96, 128, 768, 1024, _log(rng, 8, 4096), _log(rng, 8, 4096) | 1])
        return {"kind": kind, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "rows": _log(rng, 1, (64 << 20) // d),
                "d": d}
    k, n = rng.choice([(768, 2304), (768, 768), (1152, 768), (1024, 1536), (384, 1152), (2624, 1024),
                       (_log(rng, 64, 4096), _log(rng, 32, 4096)), (16 * _log(rng, 4, 256), _log(rng, 32, 4096))])
    gated = rng.random() < 0.3
    x, out = rng.choice(["bf16", "bf16", "fp16", "fp32", "int8", "int8"]), rng.choice(["bf16", "fp16", "fp32"])
    return {"kind": kind, "x": x, "out": out if x == "int8" else x,
            "rows": _log(rng, 1, min(49152, int(4e10 / (k * n * (2 if gated else 1))))), "k": k, "n": n,
            "act": rng.choice(["gelu", "gelu_tanh", "silu"]) if gated or rng.random() < 0.3 else "", "gated": gated,
            "bias": rng.random() < 0.5, "residual": rng.random() < 0.4}


# ---- inputs ---------------------------------------------------------------


def _integers(x):
    """Rows as 8-bit integers and their scales, from 64-bit quotients."""
    scale = (x.abs().amax(-1).double() / 127).float().clamp_min(2.0**-126)
    return torch.round(x.double() / scale.double()[..., None]).to(torch.int8), scale


def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    if c["kind"] == "rotary":
        dt, lead = _DT[c["dtype"]], (c["n"], c["len"])
        if c["pos"] == "packed":
            # lengths spread evenly over a sixth of the longest to it, in an order drawn from the seed
            lo = (c["len"] + 5) // 6
            lens = lo + torch.arange(c["n"], device="cuda") * (c["len"] - lo + 1) // c["n"]
            lens = lens[torch.randperm(c["n"], generator=g, device="cuda")]
            s["cu"] = torch.nn.functional.pad(lens.cumsum(0), (1, 0)).to(torch.int32)
            lead = (int(lens.sum()),)
        elif c["pos"] == "given":
            start = torch.randint(c["far"], (c["n"], 1), generator=g, device="cuda")
            s["positions"] = start + torch.arange(c["len"], device="cuda")
        i = torch.arange(c["r"] // 2, dtype=torch.float64, device="cuda")
        s["freq"] = c["base"] ** (-2.0 * i / c["r"]) / c["factor"]
        s["amp"] = 1.0 + 0.1 * math.log(c["factor"])
        # one projection makes q, k and v: rows of all heads side by side
        qkv = normal(*lead, c["h"] + 2 * c["hk"], c["d"], dtype=dt)
        s["q"], s["k"], _ = qkv.split([c["h"], c["hk"], c["hk"]], dim=-2)
        if c["train"]:
            s["q"], s["k"] = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
            s["gq"], s["gk"] = normal(*s["q"].shape, std=0.5, dtype=dt), normal(*s["k"].shape, std=0.5, dtype=dt)
    elif c["kind"] == "tokens8":
        s["x"] = normal(c["rows"], c["d"], dtype=_DT[c["dtype"]])
    else:
        rows, k, n = c["rows"], c["k"], c["n"]
        # some columns of hidden states are far larger than the others
        x = normal(rows, k) * torch.where(torch.arange(k, device="cuda") % 61 == 7, 6.0, 1.0)
        if c["x"] == "int8":
            s["x"], s["xs"] = _integers(x)
        else:
            s["x"], s["xs"] = x.to(_DT[c["x"]]), None
        total = 2 * n if c["gated"] else n  # gate rows, then up rows
        s["w"], s["ws"] = _integers(normal(total, k, std=k**-0.5))
        s["b"] = normal(total, std=0.2, dtype=_DT[c["out"]]) if c["bias"] else None
        s["r"] = normal(rows, n, dtype=_DT[c["out"]]) if c["residual"] else None
    return s


# ---- one pass ---------------------------------------------------------------


def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    with torch.no_grad():
        if c["kind"] == "rotary":
            return _rotary_plain(s, c)
        if c["kind"] == "tokens8":
            x = s["x"]
            q, scale = _integers(x)
            return {"scale": scale, "values": (q.float() * scale[:, None]).to(x.dtype)}
        return _linear_plain(s, c)


def _run_own(s, c):
    pkg = os.path.abspath("late-interaction-kernels_amd")  # the package of the tree this runs in
    if pkg not in sys.path:
        sys.path.insert(1, pkg)
    from late_interaction_kernels import encoder

    if c["kind"] == "rotary":
        q, k = encoder.rotary(s["q"], s["k"], frequencies=s["freq"], positions=s.get("positions"),
                              cu_seqlens=s.get("cu"), interleaved=c["inter"], amplitude=s["amp"])
        if not c["train"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if c["kind"] == "tokens8":
        q, scale = encoder.quantize_int8_per_token(s["x"])
        return {"scale": scale, "values": encoder.dequantize_int8_per_token(q, scale, dtype=s["x"].dtype)}
    return {"out": encoder.linear_int8(s["x"], s["w"], s["ws"], s["b"], s["r"], x_scale=s["xs"],
                                       activation=c["act"] or None, gated=c["gated"], out_dtype=_DT[c["out"]])}


def _rotary_plain(s, c):
    """(a, b) -> (a cos - b sin, b cos + a sin) of each pair, the rest of the head as it is."""
    if c["pos"] == "packed":
        cu, at = s["cu"].long(), torch.arange(s["q"].shape[0], device="cuda")
        pos = at - cu[torch.searchsorted(cu, at, right=True) - 1]
    else:
        pos = s["positions"] if c["pos"] == "given" else torch.arange(c["len"], device="cuda").expand(c["n"], -1)
    angle = pos[..., None].double() * s["freq"]
    cos, sin = ((f(angle) * s["amp"]).float()[..., None, :] for f in (torch.cos, torch.sin))
    r = c["r"]

    def turn(x, sign):
        y = x.float()
        y, rest = y[..., :r], y[..., r:]
        a, b = (y[..., 0::2], y[..., 1::2]) if c["inter"] else y.chunk(2, -1)
        a, b = a * cos - b * sin * sign, b * cos + a * sin * sign
        y = torch.stack([a, b], -1).flatten(-2) if c["inter"] else torch.cat([a, b], -1)
        return torch.cat([y, rest], -1).to(x.dtype)

    res = {"q": turn(s["q"], 1.0), "k": turn(s["k"], 1.0)}
    if c["train"]:
        res.update(dq=turn(s["gq"], -1.0), dk=turn(s["gk"], -1.0))
    return res


def _act(x, act):
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(x * 0.5**0.5))
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh((2 / math.pi) ** 0.5 * (x + 0.044715 * x * x * x)))
    return x / (1.0 + torch.exp(-x)) if act else x


def _linear_plain(s, c):
    """act(sx sw sum_k x w + b) (times the up half) + residual."""
    x, xs = (s["x"], s["xs"]) if c["x"] == "int8" else _integers(s["x"])
    wide = torch.float64 if c["out"] == "fp32" else torch.float32  # sums past 2^24 lose what 32-bit outputs show
    y = (x.to(wide) @ s["w"].to(wide).t()).float() * xs[:, None] * s["ws"]
    if c["bias"]:
        y = y + s["b"].float()
    if c["gated"]:
        gate, up = y.chunk(2, -1)
        y = _act(gate, c["act"]) * up
    else:
        y = _act(y, c["act"])
    if c["residual"]:
        y = y + s["r"].float()
    return {"out": y.to(_DT[c["out"]])}


# ---- what a pass cannot do without ------------------------------------------


def work(case):
    """Every input read once, every output written once; the index keeps its
    integers, so they are written, and read for the way back."""
    c = case
    if c["kind"] == "rotary":
        tokens = c["n"] * c["len"]
        if c["pos"] == "packed":
            lo = (c["len"] + 5) // 6
            tokens = sum(lo + i * (c["len"] - lo + 1) // c["n"] for i in range(c["n"]))
        heads, ways = tokens * (c["h"] + c["hk"]), 2 if c["train"] else 1
        return {"bytes": ways * heads * c["d"] * 2 * _EB[c["dtype"]] + (8 * tokens if c["pos"] == "given" else 0),
                "flops": ways * heads * c["r"] * 3.0}
    if c["kind"] == "tokens8":
        m = c["rows"] * c["d"]
        return {"bytes": m * (2 * _EB[c["dtype"]] + 2) + 8 * c["rows"], "flops": 4.0 * m}
    m, k, n = c["rows"], c["k"], c["n"]
    total = 2 * n if c["gated"] else n
    e = _EB[c["out"]]
    b = m * k * _EB[c["x"]] + (4 * m if c["x"] == "int8" else 0) + total * (k + 4) + m * n * e
    return {"bytes": b + (total * e if c["bias"] else 0) + (m * n * e if c["residual"] else 0),
            "flops": 2.0 * m * k * total}


# ---- 64-bit results -----------------------------------------------------------


def exact(case, seed):
    c, s = case, prepare(case, seed)
    with torch.no_grad():
        if c["kind"] == "rotary":
            return _rotary_exact(s, c)
        if c["kind"] == "tokens8":
            units, scale = _units64(s["x"].double())
            return {"scale": s["x"].double().abs().amax(1) / 127, "values": units * scale}
        return _linear_exact(s, c)


def _units64(x):
    """Whole multiples of the row's stored scale (a 32-bit number) nearest to x, ties to even."""
    scale = torch.linalg.vector_norm(x, math.inf, dim=-1, keepdim=True).div(127.0).to(torch.float32).double()
    return (x / scale).round(), scale


def _rotary_exact(s, c):
    """As products of complex numbers."""
    if c["pos"] == "packed":
        lens = s["cu"].diff().tolist()
        pos = torch.cat([torch.arange(m, device="cuda") for m in lens]).double()
    elif c["pos"] == "given":
        pos = s["positions"].double()
    else:
        pos = torch.arange(c["len"], device="cuda", dtype=torch.float64).repeat(c["n"], 1)
    theta = pos.unsqueeze(-1) * s["freq"]
    unit = torch.polar(torch.full_like(theta, s["amp"]), theta).unsqueeze(-2)
    half = c["r"] // 2

    def apply(x, by):
        y = x.detach().double().clone()
        if c["inter"]:
            z = torch.view_as_complex(y[..., :2 * half].unflatten(-1, (half, 2)).contiguous()) * by
            y[..., :2 * half] = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(y[..., :half], y[..., half:2 * half]) * by
            y[..., :half], y[..., half:2 * half] = z.real, z.imag
        return y

    res = {"q": apply(s["q"], unit), "k": apply(s["k"], unit)}
    if c["train"]:
        res["dq"], res["dk"] = apply(s["gq"], unit.conj()), apply(s["gk"], unit.conj())
    return res


def _linear_exact(s, c):
    if c["x"] == "int8":
        x = s["x"].double() * s["xs"].double().unsqueeze(1)
    else:
        units, scale = _units64(s["x"].double())
        x = units * scale
    y = x @ (s["w"].double() * s["ws"].double().unsqueeze(1)).t()
    if c["bias"]:
        y += s["b"].double()
    n = c["n"]
    gate = y[:, :n]
    if c["act"] == "gelu":
        a = gate * 0.5 * torch.special.erfc(-gate / math.sqrt(2))
    elif c["act"] == "gelu_tanh":
        a = gate * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate**3))
    elif c["act"] == "silu":
        a = gate * torch.sigmoid(gate)
    else:
        a = gate
    if c["gated"]:
        a = a * y[:, n:]
    return {"out": a + s["r"].double() if c["residual"] else a}
