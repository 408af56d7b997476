"""``layer_norm``: layer norm of token vectors with an optional residual sum, differentiable.

With a residual the sum is rounded to the type of ``x`` first: that tensor is
returned next to the result (the next residual connection reads it), and it is what
is normalised. The row's mean, variance and the gradients' sums are fp32.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _rows(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``x`` as ``[rows, d]`` with a contiguous last dim (a view where its strides allow one) and the row stride."""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    rs, cs = x2.stride()
    if cs != 1 and x2.shape[1] > 1:
        x2 = x2.contiguous()
        rs = x2.stride(0)
    return x2, rs


def _forward(x, weight, bias, residual, eps, want_stats):
    x2, xs = _rows(x)
    rows, d = x2.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    total = stats = None
    r2, rs = None, 0
    if residual is not None:
        r2, rs = _rows(residual)
        total = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if want_stats:
        stats = torch.empty(rows, 2, dtype=torch.float32, device=x.device)
    if rows:
        with _lib.on_device(x.device):
            rc = _lib.load().lik_layer_norm(
                x2.data_ptr(), xs, _lib.ptr(r2), rs, _lib.DTYPE_CODE[x.dtype], rows, d, weight.data_ptr(),
                _lib.ptr(bias), _lib.DTYPE_CODE[weight.dtype], eps, y.data_ptr(), _lib.ptr(total), _lib.ptr(stats),
                _lib.stream_of(x))
        _lib.check(rc, "lik_layer_norm")
    return y, total, stats


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        w = weight.contiguous()
        y, total, stats = _forward(x, w, None if bias is None else bias.contiguous(), residual, eps, True)
        ctx.save_for_backward(x if total is None else total, w, stats)
        ctx.has_bias = bias is not None
        ctx.set_materialize_grads(False)
        return y if total is None else (y, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gs=None):
        s, w, stats = ctx.saved_tensors
        need_x = ctx.needs_input_grad[0] or ctx.needs_input_grad[3]
        need_w, need_b = ctx.needs_input_grad[1], ctx.has_bias and ctx.needs_input_grad[2]
        if gy is None:  # only the sum was used
            return (gs if ctx.needs_input_grad[0] else None, torch.zeros_like(w) if need_w else None,
                    torch.zeros_like(w) if need_b else None, gs if ctx.needs_input_grad[3] else None, None)
        s2, ss = _rows(s)
        g2, gys = _rows(gy)
        t2, gss = (None, 0) if gs is None else _rows(gs)
        rows, d = s2.shape
        gx = torch.empty(s.shape, dtype=s.dtype, device=s.device)
        gw = torch.empty_like(w) if need_w else None
        gb = torch.empty_like(w) if need_b else None
        if rows == 0:
            for t in (gw, gb):
                if t is not None:
                    t.zero_()
        else:
            lib = _lib.load()
            code = _lib.DTYPE_CODE[s.dtype]
            nbytes = lib.lik_layer_norm_backward_workspace_size(code, rows, d)
            ws = _lib.workspace(nbytes, s.device)
            with _lib.on_device(s.device):
                rc = lib.lik_layer_norm_backward(
                    g2.data_ptr(), gys, _lib.ptr(t2), gss, s2.data_ptr(), ss, stats.data_ptr(), code, rows, d,
                    w.data_ptr(), _lib.DTYPE_CODE[w.dtype], gx.data_ptr(), _lib.ptr(gw), _lib.ptr(gb), _lib.ptr(ws),
                    nbytes, _lib.stream_of(s))
            _lib.check(rc, "lik_layer_norm_backward")
        return (gx if need_x and ctx.needs_input_grad[0] else None, gw, gb,
                gx if need_x and ctx.needs_input_grad[3] else None, None)


def layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    *,
    eps: float = 1e-5,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Layer norm over the last dimension of ``x [..., d]``.

    Args:
        x: fp16 / bf16 / fp32, ``d`` at most 8192; any row stride.
        weight, bias: ``[d]`` in the type of ``x`` or fp32 (both alike); ``bias`` may be None.
        residual: same shape and type as ``x``; added before the norm.

    Returns:
        ``y`` of the shape and type of ``x``, or ``(y, x + residual)``.
    """
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., d] with d >= 1; got {tuple(x.shape)}")
    d = x.shape[-1]
    if x.dtype not in _DTYPES:
        raise TypeError(f"layer_norm takes fp16 / bf16 / fp32; got {x.dtype}")
    if d > 8192:
        raise ValueError(f"layer_norm takes rows of at most 8192 elements; got {d}")
    if weight.shape != (d,):
        raise ValueError(f"weight must be [{d}]; got {tuple(weight.shape)}")
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"weight must have the type of x ({x.dtype}) or be fp32; got {weight.dtype}")
    if bias is not None and (bias.shape != (d,) or bias.dtype != weight.dtype):
        raise ValueError(f"bias must be [{d}] of the weight's type; got {tuple(bias.shape)} {bias.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must match x ({tuple(x.shape)}, {x.dtype}); got {tuple(residual.shape)}, "
                         f"{residual.dtype}")
    device = x.device
    if (weight.device != device or (bias is not None and bias.device != device)
            or (residual is not None and residual.device != device)):
        raise ValueError("x, weight, bias and residual must be on the same device.")
    _lib.require_gpu(x)
    if _lib.differentiates(x, weight, bias, residual):
        return _LayerNormFn.apply(x, weight, bias, residual, float(eps))
    y, total, _ = _forward(x, weight.contiguous(), None if bias is None else bias.contiguous(), residual, float(eps),
                           False)
    return y if total is None else (y, total)


__all__ = ["layer_norm"]
