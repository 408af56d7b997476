"""``gated_ffn``: the gated feed-forward block of an encoder layer, differentiable.

``y = (act(x Wg^T) * (x Wu^T)) Wo^T + residual``. Both projections, the
activation and the product are one kernel, the output projection with the residual
is a second; the backward pass is three matrix products of the same tile kernel
(one of them turns the gradient of the product into those of both projections
in its epilogue) and a sum of the weight gradients' splits in a fixed order.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _lib

ACTIVATIONS = {"gelu": 0, "gelu_tanh": 1, "silu": 2}


_FAR = (1 << 21) + 1  # elements from row to row: the kernels reach 256 rows by 32-bit offsets


def _near(x2, w_in, w_out, r2):
    f = w_out.shape[1]  # w_in's up rows are that many rows away
    return (_lib.rows16(x2, 0, _FAR), _lib.rows16(w_in, 0, _FAR if f < 768 else min(_FAR, 0x7FF80000 // (f + 256))),
            _lib.rows16(w_out, 0, _FAR), None if r2 is None else _lib.rows16(r2, 0, _FAR))


def _forward(x2, w_in, w_out, r2, act, want_kept):
    rows, d = x2.shape
    f = w_out.shape[1]
    out = torch.empty(rows, d, dtype=x2.dtype, device=x2.device)
    h = torch.empty(rows, f, dtype=x2.dtype, device=x2.device)
    gu = None
    if rows:
        lib, code = _lib.load(), _lib.DTYPE_CODE[x2.dtype]
        if want_kept:
            gu = torch.empty(lib.lik_gated_ffn_kept_size(code, rows, d, f), dtype=torch.uint8, device=x2.device)
        nbytes = lib.lik_gated_ffn_workspace_size(code, rows, d, f)
        ws = _lib.workspace(nbytes, x2.device)
        with _lib.on_device(x2.device):
            rc = lib.lik_gated_ffn(
                x2.data_ptr(), x2.stride(0), code, rows, d, f, w_in.data_ptr(), w_in.stride(0), w_out.data_ptr(),
                w_out.stride(0), _lib.ptr(r2), 0 if r2 is None else r2.stride(0), act, out.data_ptr(), h.data_ptr(),
                _lib.ptr(gu), _lib.ptr(ws), nbytes, _lib.stream_of(x2))
        _lib.check(rc, "lik_gated_ffn")
    return out, h, gu


class _GatedFfnFn(torch.autograd.Function):
    """On prepared ``[rows, d]`` inputs."""

    @staticmethod
    def forward(ctx, x2, w_in, w_out, r2, act):
        x2, w_in, w_out, r2 = _near(x2, w_in, w_out, r2)
        out, h, gu = _forward(x2, w_in, w_out, r2, act, True)
        ctx.save_for_backward(x2, w_in, w_out, h, gu)
        ctx.act = act
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x2, w_in, w_out, h, gu = ctx.saved_tensors
        (rows, d), f = x2.shape, w_out.shape[1]
        need_x, need_in, need_out = ctx.needs_input_grad[:3]
        gx = torch.empty(rows, d, dtype=x2.dtype, device=x2.device) if need_x else None
        gi = torch.empty(2 * f, d, dtype=x2.dtype, device=x2.device) if need_in else None
        go = torch.empty(d, f, dtype=x2.dtype, device=x2.device) if need_out else None
        if rows == 0:
            for t in (gi, go):
                if t is not None:
                    t.zero_()
        elif need_x or need_in or need_out:
            g = _lib.rows16(grad, 0, _FAR)
            lib, code = _lib.load(), _lib.DTYPE_CODE[x2.dtype]
            nbytes = lib.lik_gated_ffn_backward_workspace_size(code, rows, d, f)
            ws = _lib.workspace(nbytes, x2.device)
            with _lib.on_device(x2.device):
                rc = lib.lik_gated_ffn_backward(
                    g.data_ptr(), g.stride(0), x2.data_ptr(), x2.stride(0), code, rows, d, f, w_in.data_ptr(),
                    w_in.stride(0), w_out.data_ptr(), w_out.stride(0), h.data_ptr(), gu.data_ptr(), ctx.act,
                    _lib.ptr(gx), _lib.ptr(gi), _lib.ptr(go), _lib.ptr(ws), nbytes, _lib.stream_of(x2))
            _lib.check(rc, "lik_gated_ffn_backward")
        return gx, gi, go, grad if ctx.needs_input_grad[3] else None, None


def gated_ffn(
    x: torch.Tensor,
    w_in: torch.Tensor,
    w_out: torch.Tensor,
    residual: torch.Tensor | None = None,
    *,
    activation: str = "gelu",
) -> torch.Tensor:
    """``(act(x Wg^T) * (x Wu^T)) w_out^T + residual``.

    Args:
        x: ``[..., d]`` fp16 / bf16.
        w_in: ``[2 hidden, d]``: the gate's rows, then the up projection's.
        w_out: ``[d, hidden]``.
        residual: shape and type of ``x``, or None.
        activation: "gelu" (erf), "gelu_tanh" or "silu".

    Returns:
        ``[..., d]`` of the type of ``x``. ``d`` and ``hidden`` are multiples of 8 in the
        kernels; other sizes are padded with zeros (a copy of the inputs per call). The
        product of both projections is held in the type of ``x``: in fp16 it is infinite past
        65504.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}; got {activation!r}")
    if x.dim() < 1 or w_in.dim() != 2 or w_out.dim() != 2:
        raise ValueError(f"x must be [..., d], w_in [2 hidden, d], w_out [d, hidden]; got {tuple(x.shape)}, "
                         f"{tuple(w_in.shape)}, {tuple(w_out.shape)}")
    d, f = x.shape[-1], w_out.shape[1]
    if d < 1 or f < 1 or w_in.shape != (2 * f, d) or w_out.shape[0] != d:
        raise ValueError(f"w_in must be [2 hidden, d={d}] and w_out [d={d}, hidden]; got {tuple(w_in.shape)} and "
                         f"{tuple(w_out.shape)}")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"gated_ffn takes fp16 / bf16; got {x.dtype}")
    if w_in.dtype != x.dtype or w_out.dtype != x.dtype:
        raise TypeError(f"w_in and w_out must have the type of x ({x.dtype}); got {w_in.dtype} and {w_out.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must match x ({tuple(x.shape)}, {x.dtype}); got {tuple(residual.shape)}, "
                         f"{residual.dtype}")
    if w_in.device != x.device or w_out.device != x.device or (residual is not None and residual.device != x.device):
        raise ValueError("x, w_in, w_out and residual must be on the same device.")
    _lib.require_gpu(x)
    act = ACTIVATIONS[activation]
    x2, r2 = x, residual
    if x.dim() != 2:
        x2 = x.reshape(-1, d)
        r2 = None if residual is None else residual.reshape(-1, d)
    pd, pf = -d % 8, -f % 8
    if pd or pf:  # zero rows and columns add nothing to any product
        x2 = F.pad(x2, (0, pd))
        r2 = None if r2 is None else F.pad(r2, (0, pd))
        w_in = F.pad(w_in.unflatten(0, (2, f)), (0, pd, 0, pf)).reshape(2 * (f + pf), d + pd)
        w_out = F.pad(w_out, (0, pf, 0, pd))
    if _lib.differentiates(x, w_in, w_out, residual):
        out = _GatedFfnFn.apply(x2, w_in, w_out, r2, act)
    else:
        out, _, _ = _forward(*_near(x2, w_in, w_out, r2), act, False)
    if pd:
        out = out[:, :d]
    return out if x.dim() == 2 else out.reshape(x.shape)


__all__ = ["gated_ffn"]
