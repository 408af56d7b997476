"""Operators of the transformer encoder whose token vectors MaxSim scores.

Attention over padded and packed sequences, layer norm and the gated
feed-forward block, each forward and with its gradients: the layers in front
of the projection head when a late-interaction model is trained, when a corpus
is encoded and when one query is. ``run`` computes a case in its plain form
(elementary torch operations in 32 bits, rounded once at the end) or, with
``own`` set, through ``late_interaction_kernels.encoder``.

``listed`` names twelve cases, ``draw`` gives another of the same ranges,
``prepare`` makes what a program holds before the call, ``run`` is the call,
``exact`` the same outputs in 64-bit floating point.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EB = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # Encoding one user query of 32 tokens: one layer's attention, where
        # the latency of the call counts.
        {"name": "attend_query", "kind": "attend", "dtype": "bf16", "n": 1, "lq": 32, "lk": 32, "lo": 32, "h": 12,
         "hk": 12, "d": 64, "causal": False, "window": 0, "train": False},
        # One token per text over a long document's keys: the last layer of a
        # model that keeps the first token only. Grouped heads.
        {"name": "attend_one_token", "kind": "attend", "dtype": "fp16", "n": 4, "lq": 1, "lk": 8192, "lo": 5000,
         "h": 16, "hk": 4, "d": 128, "causal": False, "window": 0, "train": False},
        # Encoding a batch of padded passages of 50 to 300 tokens.
        {"name": "attend_passages", "kind": "attend", "dtype": "bf16", "n": 256, "lq": 300, "lk": 300, "lo": 50,
         "h": 12, "hk": 12, "d": 64, "causal": False, "window": 0, "train": False},
        # Encoding packed passages and long documents in a layer whose tokens
        # see 64 neighbours on each side.
        {"name": "attend_packed_window", "kind": "packed", "dtype": "fp16", "n": 48, "lo": 16, "hi": 2048, "h": 12,
         "hk": 12, "d": 64, "causal": False, "window": 64, "train": False},
        # Training step on padded passages.
        {"name": "attend_train_passages", "kind": "attend", "dtype": "bf16", "n": 128, "lq": 300, "lk": 300, "lo": 50,
         "h": 12, "hk": 12, "d": 64, "causal": False, "window": 0, "train": True},
        # Training step on page images of 1030 patches and a causal model with
        # wide, shared heads.
        {"name": "attend_train_pages", "kind": "packed", "dtype": "bf16", "n": 16, "lo": 1030, "hi": 1030, "h": 16,
         "hk": 4, "d": 128, "causal": True, "window": 0, "train": True},
        # Layer norm of one query's tokens: a launch and little else.
        {"name": "norm_query", "kind": "norm", "dtype": "bf16", "rows": 32, "d": 768, "w32": False, "bias": True,
         "residual": False, "train": False},
        # Residual sum and layer norm in a training step under autocast
        # (16-bit activations, 32-bit parameters), 128 passages.
        {"name": "norm_train_residual", "kind": "norm", "dtype": "bf16", "rows": 38400, "d": 768, "w32": True,
         "bias": True, "residual": True, "train": True},
        # Layer norm in full precision, rows of an odd length, training.
        {"name": "norm_train_fp32", "kind": "norm", "dtype": "fp32", "rows": 32961, "d": 1027, "w32": True,
         "bias": False, "residual": False, "train": True},
        # Feed-forward block of one query's tokens: every weight is read for
        # 32 rows.
        {"name": "ffn_query", "kind": "ffn", "dtype": "bf16", "rows": 32, "d": 768, "f": 1152, "act": "gelu",
         "residual": True, "train": False},
        # Feed-forward block of the valid tokens of 256 passages, encoding.
        {"name": "ffn_passages", "kind": "ffn", "dtype": "fp16", "rows": 44801, "d": 768, "f": 1152, "act": "gelu",
         "residual": True, "train": False},
        # Training step of a wide block on 16 page images.
        {"name": "ffn_train_pages", "kind": "ffn", "dtype": "bf16", "rows": 16480, "d": 1024, "f": 2816, "act": "silu",
         "residual": True, "train": True},
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n if n < 2048 else n - 1 + n % 2  # long ones are odd: no whole tiles


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "packed", "packed", "norm", "norm", "ffn", "ffn", "ffn"])
    half, train = rng.choice(["bf16", "bf16", "fp16"]), rng.random() < 0.5
    if kind in ("attend", "packed"):
        h, hk, d = rng.choice([(12, 12, 64), (16, 16, 64), (12, 4, 64), (6, 6, 32), (16, 16, 72), (16, 4, 128),
                               (8, 8, 96)])
        window = rng.choice([0, 0, rng.randint(8, 128)])
        causal = rng.random() < 0.3
        # the scores of a whole batch are kept in 32 bits by the plain form
        most = 3e8 if train else 6e8
        if kind == "packed":
            hi = _log(rng, 24, 2048 if train else 4096)
            n = max(1, min(_log(rng, 1, 256), int(most / (h * hi * hi))))
            return {"kind": kind, "dtype": half, "n": n, "lo": rng.randint(8, min(hi, 64)), "hi": hi, "h": h, "hk": hk,
                    "d": d, "causal": causal, "window": window, "train": train}
        if not train and rng.random() < 0.3:  # few new rows over many keys
            lk = _log(rng, 64, 16384)
            return {"kind": kind, "dtype": half, "n": rng.randint(1, 16), "lq": rng.choice([1, 1, rng.randint(2, 16)]),
                    "lk": lk, "lo": rng.randint(lk // 2, lk), "h": h, "hk": hk, "d": d, "causal": False, "window": 0,
                    "train": False}
        length = _log(rng, 8 if train else 1, 2048 if train else 4096)
        n = max(1, min(_log(rng, 1, 256), int(most / (h * length * length))))
        return {"kind": kind, "dtype": half, "n": n, "lq": length, "lk": length,
                "lo": rng.randint((length + 3) // 4, length), "h": h, "hk": hk, "d": d, "causal": causal,
                "window": window, "train": train}
    if kind == "norm":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        d = rng.choice([768, 1024, _log(rng, 32, 4096), _log(rng, 32, 4096) | 1])
        return {"kind": kind, "dtype": dtype, "rows": _log(rng, 1, min(65536, (48 << 20) // d)), "d": d,
                "w32": dtype == "fp32" or rng.random() < 0.5, "bias": rng.random() < 0.5,
                "residual": rng.random() < 0.5, "train": train}
    d, f = rng.choice([(768, 1152), (1024, 2624), (384, 1024), (768, 2048), (8 * _log(rng, 16, 128),
                                                                           8 * _log(rng, 32, 352))])
    return {"kind": kind, "dtype": half, "rows": _log(rng, 16 if train else 1, 16384 if train else 49152), "d": d,
            "f": f, "act": rng.choice(["gelu", "gelu", "gelu_tanh", "silu"]), "residual": rng.random() < 0.5,
            "train": train}


# ---- inputs ---------------------------------------------------------------


def _lens(n, lo, hi, g):
    """Lengths spread evenly over lo .. hi, in an order drawn from the seed
    (every seed has the same total, so outputs keep their shapes)."""
    return (lo + torch.arange(n, device="cuda") * (hi - lo + 1) // n)[torch.randperm(n, generator=g, device="cuda")]


def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[c["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    s = {"case": c}
    if c["kind"] in ("attend", "packed"):
        h, hk, d = c["h"], c["hk"], c["d"]
        if c["kind"] == "packed":
            lens = _lens(c["n"], c["lo"], c["hi"], g)
            s["cu"] = torch.nn.functional.pad(lens.cumsum(0), (1, 0)).to(torch.int32)
            lead = (int(lens.sum()),)
        else:
            lens = _lens(c["n"], c["lo"], c["lk"], g)
            s["keep"] = torch.arange(c["lk"], device="cuda")[None] < lens[:, None]
            lead = (c["n"], c["lk"])
        # one projection makes q, k and v: rows of all heads side by side
        qkv = normal(*lead, h + 2 * hk, d)
        s["q"], s["k"], s["v"] = qkv.split([h, hk, hk], dim=-2)
        s["q"] = (s["q"].float() * 1.5).to(dt) if c["train"] else s["q"]
        if c["kind"] == "attend" and c["lq"] != c["lk"]:  # a few rows of their own over the keys
            s["q"] = normal(c["n"], c["lq"], h, d, std=1.5)
        names = ("q", "k", "v")
        if c["train"]:
            s["g"] = normal(*s["q"].shape, std=0.5)
    elif c["kind"] == "norm":
        s["x"] = (torch.randn(c["rows"], c["d"], generator=g, device="cuda") * 1.7 + 0.3).to(dt)
        wt = torch.float32 if c["w32"] else dt
        s["w"] = (torch.randn(c["d"], generator=g, device="cuda") * 0.1 + 1).to(wt)
        s["b"] = normal(c["d"], std=0.1, dtype=wt) if c["bias"] else None
        s["r"] = normal(c["rows"], c["d"], std=1.2) if c["residual"] else None
        names = ("x", "w") + (("b",) if c["bias"] else ()) + (("r",) if c["residual"] else ())
        if c["train"]:
            s["g"] = normal(c["rows"], c["d"], std=0.5)
            s["gs"] = normal(c["rows"], c["d"], std=0.5) if c["residual"] else None
    else:
        rows, d, f = c["rows"], c["d"], c["f"]
        s["x"] = normal(rows, d)
        s["w_in"] = normal(2 * f, d, std=d**-0.5)  # gate rows, then up rows
        s["w_out"] = normal(d, f, std=f**-0.5)
        s["r"] = normal(rows, d) if c["residual"] else None
        names = ("x", "w_in", "w_out")
        if c["train"]:
            s["g"] = normal(rows, d, std=0.5)
    s["names"] = names
    if c["train"]:
        for k in names:
            s[k] = s[k].detach().requires_grad_()
    return s


# ---- one pass ---------------------------------------------------------------


def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    with torch.no_grad():
        if c["kind"] == "norm":
            return _norm_plain(s, c)
        if c["kind"] == "ffn":
            return _ffn_plain(s, c)
        return _attend_plain(s, c)


def _run_own(s, c):
    pkg = os.path.abspath("late-interaction-kernels_amd")  # the package of the tree this runs in
    if pkg not in sys.path:
        sys.path.insert(1, pkg)
    from late_interaction_kernels import encoder

    if c["kind"] == "attend":
        qm = s["keep"] if c["lq"] == c["lk"] else None
        out = encoder.attention(s["q"], s["k"], s["v"], qm, s["keep"], causal=c["causal"],
                                window=c["window"] or None)
    elif c["kind"] == "packed":
        out = encoder.attention_varlen(s["q"], s["k"], s["v"], s["cu"], s["cu"], c["hi"], c["hi"],
                                       causal=c["causal"], window=c["window"] or None)
    elif c["kind"] == "norm":
        out = encoder.layer_norm(s["x"], s["w"], s["b"], s["r"], eps=1e-5)
        y, total = out if c["residual"] else (out, None)
        res = {"y": y} if total is None else {"y": y, "sum": total}
        if c["train"]:
            outs, gs = ((y,), (s["g"],)) if total is None else ((y, total), (s["g"], s["gs"]))
            grads = torch.autograd.grad(outs, [s[k] for k in s["names"]], gs)
            res.update(("d" + k, x) for k, x in zip(s["names"], grads))
        return res
    else:
        out = encoder.gated_ffn(s["x"], s["w_in"], s["w_out"], s["r"], activation=c["act"])
    if not c["train"]:
        return {"out": out}
    grads = torch.autograd.grad(out, [s[k] for k in s["names"]], s["g"])
    return {"out": out, **{"d" + k: x for k, x in zip(s["names"], grads)}}


def _visible(c, lq, lk, device):
    """[lq, lk] keep flags of the causal order and the window; None where every pair is kept."""
    if not (c["causal"] or c["window"]):
        return None
    ahead = torch.arange(lk, device=device)[None] - torch.arange(lq, device=device)[:, None]
    keep = ahead <= 0 if c["causal"] else ahead <= c["window"]
    return keep & (ahead >= -c["window"]) if c["window"] else keep


def _attend_plain(s, c):
    """softmax(q k^T / sqrt(d)) v over the kept pairs, and its gradients."""
    dt = s["q"].dtype
    q, k, v, g = (None if s.get(x) is None else s[x].float() for x in ("q", "k", "v", "g"))
    if c["kind"] == "packed":  # rows to [n, hi]
        cu = s["cu"].long()
        at = torch.arange(q.shape[0], device=q.device)
        seq = torch.searchsorted(cu, at, right=True) - 1
        place = seq * c["hi"] + at - cu[seq]
        keep = torch.zeros(c["n"] * c["hi"], dtype=torch.bool, device=q.device)
        keep[place] = True
        keep = keep.view(c["n"], c["hi"])

        def spread(x):
            y = x.new_zeros(c["n"] * c["hi"], *x.shape[1:])
            y[place] = x
            return y.view(c["n"], c["hi"], *x.shape[1:])

        q, k, v, g = (None if x is None else spread(x) for x in (q, k, v, g))
    else:
        keep = s["keep"]
    n, lq, h, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    q, g = (None if x is None else x.transpose(1, 2).contiguous() for x in (q, g))  # [n, h, lq, d]
    k, v = (x.transpose(1, 2).repeat_interleave(h // hk, 1) for x in (k, v))
    scale = d**-0.5
    pair = keep[:, None, None, :]
    if lq == lk:
        pair = pair & keep[:, None, :, None]
    seen = _visible(c, lq, lk, q.device)
    if seen is not None:
        pair = pair & seen
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    p.masked_fill_(~pair, -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, 1.0, total))
    res = {"out": torch.matmul(p, v)}
    if c["train"]:
        dv = torch.matmul(p.transpose(2, 3).contiguous(), g)
        dp = torch.matmul(g, v.transpose(2, 3).contiguous())
        ds = dp.sub_((p * dp).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
        res.update(dq=torch.matmul(ds, k), dk=dk.view(n, hk, -1, lk, d).sum(2), dv=dv.view(n, hk, -1, lk, d).sum(2))
    res = {name: x.transpose(1, 2) for name, x in res.items()}
    if c["kind"] == "packed":
        res = {name: x.reshape(-1, *x.shape[2:])[place] for name, x in res.items()}
    return {name: x.to(dt) for name, x in res.items()}


def _norm_plain(s, c):
    dt = s["x"].dtype
    x, total = s["x"].float(), None
    if c["residual"]:
        total = (x + s["r"].float()).to(dt)  # what the next layer reads is what is normalised
        x = total.float()
    w = s["w"].float()
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / ((xc * xc).mean(-1, keepdim=True) + 1e-5).sqrt()
    xh = xc * rstd
    y = xh * w if s["b"] is None else xh * w + s["b"].float()
    res = {"y": y.to(dt)} if total is None else {"y": y.to(dt), "sum": total}
    if c["train"]:
        g = s["g"].float()
        gw = g * w
        dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
        if c["residual"]:
            dx = dx + s["gs"].float()
            res["dr"] = dx.to(dt)
        res["dx"] = dx.to(dt)
        res["dw"] = (g * xh).sum(0).to(s["w"].dtype)
        if c["bias"]:
            res["db"] = g.sum(0).to(s["b"].dtype)
    return res


def _act(x, act):
    """The activation and its derivative."""
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(x * 0.5**0.5))
        return x * cdf, cdf + x * torch.exp(-0.5 * x * x) * (2 * math.pi) ** -0.5
    if act == "gelu_tanh":
        a = (2 / math.pi) ** 0.5
        t = torch.tanh(a * (x + 0.044715 * x * x * x))
        return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * a * (1 + 3 * 0.044715 * x * x)
    sig = 1.0 / (1.0 + torch.exp(-x))
    return x * sig, sig * (1 + x * (1 - sig))


def _ffn_plain(s, c):
    """y = (act(x Wg^T) * (x Wu^T)) Wo^T + residual, and its gradients."""
    dt = s["x"].dtype
    x, w_in, w_out = s["x"].float(), s["w_in"].float(), s["w_out"].float()
    gate, up = (x @ w_in.t()).chunk(2, -1)
    a, slope = _act(gate, c["act"])
    hidden = a * up
    y = hidden @ w_out.t()
    if c["residual"]:
        y = y + s["r"].float()
    res = {"out": y.to(dt)}
    if c["train"]:
        g = s["g"].float()
        dh = g @ w_out
        dgu = torch.cat([dh * up * slope, dh * a], -1)
        res.update(dx=(dgu @ w_in).to(dt), dw_in=(dgu.t() @ x).to(dt), dw_out=(g.t() @ hidden).to(dt))
    return res


# ---- what a pass cannot do without ------------------------------------------


def _near(length, left, right):
    """Pairs (i, j) of one sequence with i - left <= j <= i + right."""
    def side(m):  # pairs with 0 < j - i <= m
        m = min(m, length - 1)
        return m * length - m * (m + 1) / 2

    return length + side(left) + side(right)


def work(case):
    """Valid tokens and the pairs they keep, at lengths spread evenly; every
    input read once, every output written once. Gradients of attention take
    four products next to the forward's two, those of a linear layer two next
    to its one."""
    c = case
    e = _EB[c["dtype"]]
    if c["kind"] in ("attend", "packed"):
        h, hk, d, n = c["h"], c["hk"], c["d"], c["n"]
        hi = c["hi"] if c["kind"] == "packed" else c["lk"]
        steps = min(n, 64)
        lens = [c["lo"] + int((i + 0.5) * (hi - c["lo"] + 1) / steps) for i in range(steps)]
        lens = [min(x, hi) for x in lens]
        tokens = n * sum(lens) / steps
        if c["kind"] == "attend" and c["lq"] != c["lk"]:
            pairs, rows = c["lq"] * tokens, n * c["lq"]
        else:
            left = c["window"] or hi
            right = 0 if c["causal"] else left
            pairs, rows = n * sum(_near(x, left, right) for x in lens) / steps, tokens
        out = n * c["lq"] if c["kind"] == "attend" else rows  # rows written, padded ones among them
        keys = n * c["lk"] if c["kind"] == "attend" else tokens
        b = (rows * h + 2 * tokens * hk + out * h) * d * e + (n * hi if c["kind"] == "attend" else 4 * n)
        f = 4.0 * d * h * pairs
        if c["train"]:
            b += (rows * h + out * h + 2 * keys * hk) * d * e
            f *= 3
        return {"bytes": b, "flops": f}
    if c["kind"] == "norm":
        m = c["rows"] * c["d"]
        b = m * e * (2 + (2 if c["residual"] else 0))
        if c["train"]:
            b += m * e * (2 + (2 if c["residual"] else 0)) + 8 * c["d"]
        return {"bytes": b + 8 * c["d"], "flops": (8.0 + (12.0 if c["train"] else 0)) * m}
    m, d, f = c["rows"], c["d"], c["f"]
    b = e * (m * d * (3 if c["residual"] else 2) + 3 * d * f)
    if c["train"]:
        b += e * (2 * m * d + 3 * d * f)
    return {"bytes": b, "flops": (3 if c["train"] else 1) * 6.0 * m * d * f}


# ---- 64-bit results -----------------------------------------------------------


def exact(case, seed):
    c, s = case, prepare(case, seed)
    with torch.no_grad():
        d64 = {k: x.detach().double() for k, x in s.items()
               if isinstance(x, torch.Tensor) and x.is_floating_point()}
        if c["kind"] == "norm":
            return _norm_exact(s, d64, c)
        if c["kind"] == "ffn":
            return _ffn_exact(d64, c)
        return _attend_exact(s, d64, c)


def _attend_exact(s, x, c):
    """Sequence by sequence, the kept rows only."""
    res = {"out": torch.zeros_like(x["q"])}
    if c["train"]:
        res.update(dq=torch.zeros_like(x["q"]), dk=torch.zeros_like(x["k"]), dv=torch.zeros_like(x["v"]))
    h, hk, d = c["h"], c["hk"], c["d"]
    if c["kind"] == "packed":
        cu = s["cu"].tolist()
        spots = [(slice(a, b), slice(a, b)) for a, b in zip(cu, cu[1:])]
    else:
        lens = s["keep"].sum(1).tolist()
        spots = [((i, slice(0, m if c["lq"] == c["lk"] else c["lq"])), (i, slice(0, m))) for i, m in enumerate(lens)]
    for rows, cols in spots:
        q = x["q"][rows].transpose(0, 1)  # [h, rows, d]
        k, v = (x[t][cols].transpose(0, 1) for t in ("k", "v"))
        heads = torch.arange(h, device=q.device) * hk // h
        k, v = k[heads], v[heads]
        a = (q @ k.transpose(1, 2).contiguous()) / math.sqrt(d)
        i, j = torch.arange(a.shape[1], device=a.device)[:, None], torch.arange(a.shape[2], device=a.device)
        if c["causal"]:
            a = a.masked_fill(j > i, -math.inf)
        if c["window"]:
            a = a.masked_fill((j - i).abs() > c["window"], -math.inf)
        p = torch.exp(a - torch.logsumexp(a, -1, keepdim=True))
        o = p @ v
        res["out"][rows] = o.transpose(0, 1)
        if c["train"]:
            g = x["g"][rows].transpose(0, 1)
            ds = p * (g @ v.transpose(1, 2).contiguous() - (g * o).sum(-1, keepdim=True)) / math.sqrt(d)
            res["dq"][rows] = (ds @ k).transpose(0, 1)
            for name, left, right in (("dk", ds, q), ("dv", p, g)):
                each = left.transpose(1, 2).contiguous() @ right
                res[name][cols] = each.view(hk, h // hk, *each.shape[1:]).sum(1).transpose(0, 1)
    return res


def _norm_exact(s, x, c):
    a, res = x["x"], {}
    if c["residual"]:
        res["sum"] = a + x["r"]
        a = res["sum"].to(s["x"].dtype).double()  # the definition: the stored sum is normalised
    var, mean = torch.var_mean(a, -1, correction=0, keepdim=True)
    unit = (a - mean) * (var + 1e-5).rsqrt()
    res["y"] = unit * x["w"] + (x["b"] if c["bias"] else 0.0)
    if c["train"]:
        gw = x["g"] * x["w"]
        n = c["d"]
        back = gw - gw.sum(-1, keepdim=True) / n - unit * ((gw * unit).sum(-1, keepdim=True) / n)
        res["dx"] = back * (var + 1e-5).rsqrt()
        if c["residual"]:
            res["dx"] = res["dr"] = res["dx"] + x["gs"]
        res["dw"] = (x["g"] * unit).sum(0)
        if c["bias"]:
            res["db"] = x["g"].sum(0)
    return res


def _ffn_exact(x, c):
    f = c["f"]
    gate, up = x["x"] @ x["w_in"][:f].t(), x["x"] @ x["w_in"][f:].t()
    if c["act"] == "gelu":
        cdf = 0.5 * torch.special.erfc(-gate / math.sqrt(2))
        a, slope = gate * cdf, cdf + gate * torch.exp(-gate * gate / 2) / math.sqrt(2 * math.pi)
    elif c["act"] == "gelu_tanh":
        u = math.sqrt(2 / math.pi) * (gate + 0.044715 * gate**3)
        du = math.sqrt(2 / math.pi) * (1 + 0.134145 * gate**2)
        a = gate * torch.sigmoid(2 * u)  # (1 + tanh u) / 2
        slope = torch.sigmoid(2 * u) + 2 * gate * torch.sigmoid(2 * u) * torch.sigmoid(-2 * u) * du
    else:
        a = gate * torch.sigmoid(gate)
        slope = torch.sigmoid(gate) + a * torch.sigmoid(-gate)
    res = {"out": (a * up) @ x["w_out"].t() + (x["r"] if c["residual"] else 0.0)}
    if c["train"]:
        dh = x["g"] @ x["w_out"]
        dgate, dup = dh * up * slope, dh * a
        res["dx"] = dgate @ x["w_in"][:f] + dup @ x["w_in"][f:]
        res["dw_in"] = torch.cat([dgate.t() @ x["x"], dup.t() @ x["x"]])
        res["dw_out"] = x["g"].t() @ (a * up)
    return res
