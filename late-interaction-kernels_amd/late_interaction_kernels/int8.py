"""Token vectors and linear layers in 8-bit integers.

``quantize_int8_per_token`` / ``dequantize_int8_per_token``: rows as integers of
-127 .. 127 with an fp32 scale each, and back. ``linear_int8``: a linear layer on such rows
and a weight quantised the same way (a scale per output channel). Inference only.
"""

from __future__ import annotations

import torch

from . import _lib
from .layer_norm import _rows

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _no_gradient(what, *tensors):
    """8-bit integers carry no gradient: a call that would drop one is refused."""
    if _lib.differentiates(*tensors):
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
    if X.dim() < 1 or not 1 <= X.shape[-1] <= 1 << 24:
        raise ValueError(f"X must be [..., d] with 1 <= d <= 2^24; got {tuple(X.shape)}")
    if X.dtype not in _DTYPES:
        raise TypeError(f"quantize_int8_per_token takes fp16 / bf16 / fp32; got {X.dtype}")
    _lib.require_gpu(X)
    _no_gradient("quantize_int8_per_token", X)
    out = torch.empty(X.shape, dtype=torch.int8, device=X.device)
    scale = torch.empty(X.shape[:-1], dtype=torch.float32, device=X.device)
    if X.numel():
        d = X.shape[-1]
        x2, xs = _rows(X)
        with _lib.on_device(X.device):
            rc = _lib.load().lik_quantize_int8(x2.data_ptr(), xs, _lib.DTYPE_CODE[X.dtype], x2.shape[0], d,
                                               out.data_ptr(), d, scale.data_ptr(), _lib.stream_of(X))
        _lib.check(rc, "lik_quantize_int8")
    return out, scale


def dequantize_int8_per_token(
    X_int8: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.float32
) -> torch.Tensor:
    """``X_int8 * scale`` of each row, rounded once to ``dtype`` (fp16 / bf16 / fp32); ``scale`` is fp32
    ``X_int8.shape[:-1]``."""
    if X_int8.dtype != torch.int8 or scale.dtype != torch.float32:
        raise TypeError(f"X_int8 must be int8 and scale fp32; got {X_int8.dtype} and {scale.dtype}")
    if X_int8.dim() < 1 or not 1 <= X_int8.shape[-1] <= 1 << 24:
        raise ValueError(f"X_int8 must be [..., d] with 1 <= d <= 2^24; got {tuple(X_int8.shape)}")
    if scale.shape != X_int8.shape[:-1]:
        raise ValueError(f"scale must be {list(X_int8.shape[:-1])}; got {tuple(scale.shape)}")
    if dtype not in _DTYPES:
        raise TypeError(f"dequantize_int8_per_token gives fp16 / bf16 / fp32; got {dtype}")
    if scale.device != X_int8.device:
        raise ValueError("X_int8 and scale must be on the same device.")
    _lib.require_gpu(X_int8)
    _no_gradient("dequantize_int8_per_token", scale)
    out = torch.empty(X_int8.shape, dtype=dtype, device=X_int8.device)
    if out.numel():
        (x2, xs), scale = _rows(X_int8), scale.contiguous()
        with _lib.on_device(out.device):
            rc = _lib.load().lik_dequantize_int8(x2.data_ptr(), xs, scale.data_ptr(), _lib.DTYPE_CODE[dtype],
                                                 x2.shape[0], x2.shape[1], out.data_ptr(), _lib.stream_of(out))
        _lib.check(rc, "lik_dequantize_int8")
    return out


__all__ = ["dequantize_int8_per_token", "quantize_int8_per_token"]
