"""Token vectors and linear layers in 8-bit integers.

``quantize_int8_per_token`` / ``dequantize_int8_per_token``: rows as integers of
-127 .. 127 with an fp32 scale each, and back. ``linear_int8``: a linear layer on such rows
and a weight quantised the same way (a scale per output channel). Inference only.
"""

from __future__ import annotations

import torch

from . import _lib
from .gated_ffn import ACTIVATIONS
from .layer_norm import _rows

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _no_gradient(what, *tensors):
    """8-bit integers carry no gradient: a call that would drop one is refused."""
    if _lib.differentiates(*tensors):  # (or forward-mode differentiation is active)
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad(), or on detached tensors")


def quantize_int8_per_token(X: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Each row (last axis) as 8-bit integers with its own scale.

    ``scale = max(max|x| / 127, 2^-126)`` in fp32, ``X_int8 = x / scale`` to the nearest integer
    (of the exact quotient, ties to even), so a row of zeros stays one. A row that holds an
    infinity or a NaN gets the scale NaN and zeros: everything computed from it is NaN.

    Args:
        X: ``[..., d]`` fp16 / bf16 / fp32, any strides.

    Returns:
        ``(X_int8, scale)``: int8 of the shape of ``X`` and fp32 ``X.shape[:-1]``. A weight ``[out, in]``
        gives what :func:`linear_int8` takes.
    """
    shape, dtype = X.shape, X.dtype
    if not shape or not 1 <= shape[-1] <= 1 << 24:
        raise ValueError(f"X must be [..., d] with 1 <= d <= 2^24; got {tuple(shape)}")
    if dtype not in _DTYPES:
        raise TypeError(f"quantize_int8_per_token takes fp16 / bf16 / fp32; got {dtype}")
    _lib.require_gpu(X)
    _no_gradient("quantize_int8_per_token", X)
    out = torch.empty_like(X, dtype=torch.int8, memory_format=torch.contiguous_format)
    scale = X.new_empty(shape[:-1], dtype=torch.float32)
    x2, xs = _rows(X)
    rows, d = x2.shape
    if rows:
        device = X.device
        with _lib.on_device(device):
            rc = _lib.load().lik_quantize_int8(x2.data_ptr(), xs, _lib.DTYPE_CODE[dtype], rows, d, out.data_ptr(), d,
                                               scale.data_ptr(), _lib.stream_of(X))
        _lib.check(rc, "lik_quantize_int8")
    return out, scale


def dequantize_int8_per_token(
    X_int8: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.float32
) -> torch.Tensor:
    """``X_int8 * scale`` of each row in fp32, then rounded to ``dtype`` (fp16 / bf16 / fp32); ``scale`` is fp32
    ``X_int8.shape[:-1]``. This is how an index or hidden states held in 8 bits get
    back to the operators that read 16-bit or fp32 rows (MaxSim among them)."""
    if X_int8.dtype != torch.int8 or scale.dtype != torch.float32:
        raise TypeError(f"X_int8 must be int8 and scale fp32; got {X_int8.dtype} and {scale.dtype}")
    shape = X_int8.shape
    if not shape or not 1 <= shape[-1] <= 1 << 24:
        raise ValueError(f"X_int8 must be [..., d] with 1 <= d <= 2^24; got {tuple(shape)}")
    if scale.shape != shape[:-1]:
        raise ValueError(f"scale must be {list(shape[:-1])}; got {tuple(scale.shape)}")
    if dtype not in _DTYPES:
        raise TypeError(f"dequantize_int8_per_token gives fp16 / bf16 / fp32; got {dtype}")
    device = X_int8.device
    if scale.device != device:
        raise ValueError("X_int8 and scale must be on the same device.")
    _lib.require_gpu(X_int8)
    _no_gradient("dequantize_int8_per_token", scale)
    out = torch.empty_like(X_int8, dtype=dtype, memory_format=torch.contiguous_format)
    (x2, xs), scale = _rows(X_int8), scale if scale.is_contiguous() else scale.contiguous()
    rows, d = x2.shape
    if rows:
        with _lib.on_device(device):
            rc = _lib.load().lik_dequantize_int8(x2.data_ptr(), xs, scale.data_ptr(), _lib.DTYPE_CODE[dtype], rows, d,
                                                 out.data_ptr(), _lib.stream_of(out))
        _lib.check(rc, "lik_dequantize_int8")
    return out


_LIK_INT8 = 4
_FAR = 1 << 23  # bytes from row to row of integers: the kernels reach 256 rows by 32-bit offsets


def _integer_rows(x: torch.Tensor, zeros: bool, far: int) -> torch.Tensor:
    """``x`` with rows that start on 16 bytes and go on to a multiple of 16 (with zeros there, or with whatever the
    storage holds), less than ``far`` apart: a copy where they do not."""
    n, k = x.shape
    rs, cs = x.stride()
    if (cs == 1 or k == 1) and not (rs | x.data_ptr()) & 15 and rs < far:
        if k % 16 == 0:
            return x
        if not zeros and x.storage_offset() + (n - 1) * rs + (k + 15) // 16 * 16 <= x.untyped_storage().nbytes():
            return x
    y = torch.nn.functional.pad(x, (0, -k % 16)) if k % 16 else x.clone(memory_format=torch.contiguous_format)
    return y if y.is_contiguous() and y.data_ptr() % 16 == 0 else y.clone(memory_format=torch.contiguous_format)


def linear_int8(
    x: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    *,
    x_scale: torch.Tensor | None = None,
    activation: str | None = None,
    gated: bool = False,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """``act(x W^T + bias) + residual`` with both factors as 8-bit integers; ``gated``:
    ``act(x Wg^T + bg) * (x Wu^T + bu) + residual``.

    Args:
        x: ``[..., in]`` fp16 / bf16 / fp32, quantised per token within the call (as by
            :func:`quantize_int8_per_token`), or int8 with its ``x_scale``. ``in`` at most 131071: sums are exact.
        weight: int8 ``[out, in]`` (gated: ``[2 out, in]``, the gate's rows, then the up rows).
        weight_scale: fp32, one for each of its rows.
        bias: as many, of the output's type or fp32, or None.
        residual: ``[..., out]`` of the output's type, or None; added after the activation.
        x_scale: fp32 ``x.shape[:-1]``, for int8 ``x`` only.
        activation: None, "gelu" (erf), "gelu_tanh" or "silu".
        out_dtype: fp16 / bf16 / fp32; default the type of ``x`` (int8: bf16).

    Returns:
        ``[..., out]``, everything after the integer sums in fp32 and rounded once ("gelu" of 16-bit
        outputs is off by up to 1e-7 of its argument). ``in`` is a multiple of 16 in the kernels; a weight of another
        width (int8 ``x`` too) is padded in a copy per call, unless its rows lie a multiple of 16 bytes apart (a
        slice of a wider one).
    """
    if activation is not None and activation not in ACTIVATIONS:
        raise ValueError(f"activation must be None or one of {sorted(ACTIVATIONS)}; got {activation!r}")
    if x.dim() < 1 or weight.dim() != 2:
        raise ValueError(f"x must be [..., in] and weight [out, in]; got {tuple(x.shape)} and {tuple(weight.shape)}")
    total, k = weight.shape
    *lead, width = x.shape
    dtype, device = x.dtype, x.device
    if width != k or k < 1 or total < 1 or (gated and total % 2):
        raise ValueError(f"weight must be [{'2 out' if gated else 'out'}, in={width}]; got {tuple(weight.shape)}")
    if k > 131071:
        raise ValueError(f"linear_int8 takes at most 131071 input features; got {k}")
    n = total // 2 if gated else total
    int8 = dtype == torch.int8
    if not int8 and dtype not in _DTYPES:
        raise TypeError(f"linear_int8 takes fp16 / bf16 / fp32 / int8; got {dtype}")
    if weight.dtype != torch.int8 or weight_scale.dtype != torch.float32:
        raise TypeError(f"weight must be int8 and weight_scale fp32; got {weight.dtype} and {weight_scale.dtype}")
    if weight_scale.shape != (total,):
        raise ValueError(f"weight_scale must be [{total}]; got {tuple(weight_scale.shape)}")
    if int8 != (x_scale is not None):
        raise ValueError("x_scale goes with int8 x, and only with it")
    if int8:
        if list(x_scale.shape) != lead or x_scale.dtype != torch.float32:
            raise ValueError(f"x_scale must be fp32 {lead}; got {x_scale.dtype} {tuple(x_scale.shape)}")
        if x_scale.device != device:
            raise ValueError("x, weight, their scales, bias and residual must be on the same device.")
    out_dtype = out_dtype or (torch.bfloat16 if int8 else dtype)
    if out_dtype not in _DTYPES:
        raise TypeError(f"linear_int8 gives fp16 / bf16 / fp32; got {out_dtype}")
    if bias is not None:
        if bias.shape != (total,) or bias.dtype not in (out_dtype, torch.float32):
            raise ValueError(f"bias must be [{total}] of {out_dtype} or fp32; got {tuple(bias.shape)} {bias.dtype}")
        if bias.device != device:
            raise ValueError("x, weight, their scales, bias and residual must be on the same device.")
    if residual is not None:
        if list(residual.shape) != [*lead, n] or residual.dtype != out_dtype:
            raise ValueError(f"residual must be {[*lead, n]} of {out_dtype}; got {tuple(residual.shape)} "
                             f"{residual.dtype}")
        if residual.device != device:
            raise ValueError("x, weight, their scales, bias and residual must be on the same device.")
    if weight.device != device or weight_scale.device != device:
        raise ValueError("x, weight, their scales, bias and residual must be on the same device.")
    _lib.require_gpu(x)
    _no_gradient("linear_int8", x, weight_scale, bias, residual, x_scale)
    out = x.new_empty((*lead, n), dtype=out_dtype)
    if out.numel() == 0:
        return out
    x2, xs = _rows(x)
    x_code = _LIK_INT8
    if int8:
        x2 = _integer_rows(x2, True, _FAR)
        k, xs = x2.shape[1], x2.stride(0)
        if not x_scale.is_contiguous():
            x_scale = x_scale.contiguous()
    else:
        x_code = _lib.DTYPE_CODE[dtype]
    # (a gated weight's up rows are n rows away from the gate's)
    w = _integer_rows(weight, False, min(_FAR, 0xFFF00000 // (n + 256)) if gated else _FAR)
    if not weight_scale.is_contiguous():
        weight_scale = weight_scale.contiguous()
    b_ptr = r_ptr = rs = b_code = 0
    if bias is not None:
        if not bias.is_contiguous():
            bias = bias.contiguous()
        b_ptr, b_code = bias.data_ptr(), _lib.DTYPE_CODE[bias.dtype]
    if residual is not None:
        r2, rs = _rows(residual)
        r_ptr = r2.data_ptr()
    a = _lib.pack_linear_int8(
        x2.data_ptr(), x_scale.data_ptr() if int8 else 0, w.data_ptr(), weight_scale.data_ptr(), b_ptr, r_ptr, xs,
        w.stride(0), rs, x2.shape[0], k, n, x_code, _lib.DTYPE_CODE[out_dtype], b_code,
        -1 if activation is None else ACTIVATIONS[activation], gated)
    lib = _lib.load()
    nbytes = lib.lik_linear_int8_workspace_size(a)
    ws = _lib.workspace(nbytes, device)
    with _lib.on_device(device):
        rc = lib.lik_linear_int8(a, out.data_ptr(), _lib.ptr(ws), nbytes, _lib.stream_of(x))
    _lib.check(rc, "lik_linear_int8")
    return out


__all__ = ["dequantize_int8_per_token", "linear_int8", "quantize_int8_per_token"]
