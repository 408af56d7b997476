"""The encoder operators in 64 bits, from their formulas, and the measure their tests use."""

from __future__ import annotations

import math

import torch

# unit roundoff of the 16-bit types: a result rounded once is off by at most this share of itself
ROUNDOFF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def off(got: torch.Tensor, want: torch.Tensor) -> float:
    """2-norm of the difference over the 2-norm of the result (0 / 0 = 0)."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.isfinite(got).all()
    d, n = float((got - want).norm()), float(want.norm())
    return 0.0 if d == 0 else d / n if n else math.inf


def layer_norm64(x, w, b, r, eps, dtype):
    """``(y, sum)`` with the sum rounded to ``dtype``, as the operator defines it."""
    total = x if r is None else (x + r).to(dtype).double() if dtype is not None else x + r
    mean = total.mean(-1, keepdim=True)
    var = ((total - mean) ** 2).mean(-1, keepdim=True)
    y = (total - mean) / torch.sqrt(var + eps) * w
    return (y if b is None else y + b), total


def act64(x, name):
    if name == "gelu":
        return 0.5 * x * (1 + torch.erf(x / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x**3)))
    return x * torch.sigmoid(x)


def gated_ffn64(x, w_in, w_out, r, name):
    f = w_out.shape[1]
    y = (act64(x @ w_in[:f].t(), name) * (x @ w_in[f:].t())) @ w_out.t()
    return y if r is None else y + r


def keep_pairs(lq, lk, causal, window):
    j, i = torch.arange(lk)[None], torch.arange(lq)[:, None]
    keep = torch.ones(lq, lk, dtype=torch.bool)
    if causal:
        keep &= j <= i
    if window is not None:
        keep &= (j - i).abs() <= window
    return keep


def attention64(q, k, v, keep, scale):
    """``q [lq, H, d]``, ``k, v [lk, Hk, d]``, ``keep [lq, lk]`` of one sequence; rows that
    keep nothing are zeros, rows of k and v that nothing keeps are not touched."""
    g = q.shape[1] // k.shape[1]
    used = keep.any(0)
    k = torch.where(used[:, None, None], k, torch.zeros((), dtype=k.dtype))
    v = torch.where(used[:, None, None], v, torch.zeros((), dtype=v.dtype))
    q = torch.where(keep.any(1)[:, None, None], q, torch.zeros((), dtype=q.dtype))
    kk, vv = k.repeat_interleave(g, 1).transpose(0, 1), v.repeat_interleave(g, 1).transpose(0, 1)
    s = scale * q.transpose(0, 1) @ kk.transpose(1, 2)
    top = torch.where(keep, s, torch.tensor(-math.inf, dtype=s.dtype)).amax(-1, keepdim=True).detach()
    p = torch.where(keep, torch.exp(torch.where(keep, s - torch.where(top.isinf(), 0.0, top), 0.0)), 0.0)
    total = p.sum(-1, keepdim=True)
    return ((p / torch.where(total == 0, 1.0, total)) @ vv).transpose(0, 1)
