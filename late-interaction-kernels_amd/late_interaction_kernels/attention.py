"""``attention`` / ``attention_varlen``: softmax attention of token sequences, padded
or packed, differentiable.

One pass over the keys with the running maximum and sum of the softmax; the
scores never reach memory. Few queries over long keys are split over the keys and
joined. The backward pass computes the probabilities again from one kept
statistic per query and head, and sums every gradient in a fixed order (no
atomics). Query heads may share key / value heads (``H`` a multiple of ``Hk``).
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._core import _i32, _mask_i8, assert_max_seqlens_cover, seqlen_max


_FAR = 1 << 24  # elements from token to token: the kernels reach 64 tokens by 32-bit offsets


def _args(q, k, v, meta, qm, km, cu_q, cu_k):
    """The C struct of a call on prepared ``[n, L, H, d]`` (packed: ``[T, H, d]``) tensors."""
    left, right, scale, max_q, max_k = meta
    code = _lib.DTYPE_CODE[q.dtype]
    if cu_q is not None:
        (qr, h, d), (kr, hk, _) = q.shape, k.shape
        (ql, qh, _), (kl, kh, _), (vl, vh, _) = q.stride(), k.stride(), v.stride()
        return _lib.LikAttention(q.data_ptr(), k.data_ptr(), v.data_ptr(), code, h, hk, d, cu_q.numel() - 1, max_q,
                                 max_k, 0, ql, qh, 0, kl, kh, 0, vl, vh, cu_q.data_ptr(), cu_k.data_ptr(), qr, kr,
                                 None, 0, 0, None, 0, 0, left, right, scale)
    (n, lq, h, d), (_, lk, hk, _) = q.shape, k.shape
    (qn, ql, qh, _), (kn, kl, kh, _), (vn, vl, vh, _) = q.stride(), k.stride(), v.stride()
    qmn, qml = (0, 0) if qm is None else qm.stride()
    kmn, kml = (0, 0) if km is None else km.stride()
    return _lib.LikAttention(q.data_ptr(), k.data_ptr(), v.data_ptr(), code, h, hk, d, n, lq, lk, qn, ql, qh, kn, kl, kh,
                             vn, vl, vh, None, None, 0, 0, _lib.ptr(qm), qmn, qml, _lib.ptr(km), kmn, kml, left, right,
                             scale)


def _forward(q, k, v, meta, qm, km, cu_q, cu_k, train):
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    rows = q.numel() // (q.shape[-1] * q.shape[-2])
    lse = torch.empty(q.shape[-2], rows, dtype=torch.float32, device=q.device) if train else None
    low = torch.empty(q.shape, dtype=torch.int8, device=q.device) if train else None
    if q.numel() == 0:
        return out, lse, low
    a = _args(q, k, v, meta, qm, km, cu_q, cu_k)
    if a.n == 0 or a.q_len == 0:  # packed rows in no sequence
        return out.zero_(), lse, low
    lib = _lib.load()
    nbytes = lib.lik_attention_workspace_size(ctypes.byref(a))
    ws = _lib.workspace(nbytes, q.device)
    with _lib.on_device(q.device):
        rc = lib.lik_attention(ctypes.byref(a), out.data_ptr(), _lib.ptr(lse), _lib.ptr(low), _lib.ptr(ws),
                               nbytes, _lib.stream_of(q))
    _lib.check(rc, "lik_attention")
    return out, lse, low


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, meta, qm, km, cu_q, cu_k):
        q, k, v = _lib.rows16(q, -3, _FAR), _lib.rows16(k, -3, _FAR), _lib.rows16(v, -3, _FAR)
        out, lse, low = _forward(q, k, v, meta, qm, km, cu_q, cu_k, True)
        ctx.save_for_backward(q, k, v, out, lse, low, qm, km, cu_q, cu_k)
        ctx.meta = meta
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, out, lse, low, qm, km, cu_q, cu_k = ctx.saved_tensors
        need_q, need_k, need_v = ctx.needs_input_grad[:3]
        a = _args(q, k, v, ctx.meta, qm, km, cu_q, cu_k)
        none = q.numel() == 0 or a.n == 0 or a.q_len == 0 or a.k_len == 0
        make = torch.zeros if none else torch.empty
        gq = make(q.shape, dtype=q.dtype, device=q.device) if need_q else None
        gk = gv = None
        if need_k or need_v:
            gk, gv = (make(t.shape, dtype=t.dtype, device=t.device) for t in (k, v))
        if not none and (gq is not None or gk is not None):
            g = _lib.rows16(grad, -3, _FAR)
            lib = _lib.load()
            nbytes = lib.lik_attention_backward_workspace_size(ctypes.byref(a))
            ws = _lib.workspace(nbytes, q.device)
            with _lib.on_device(q.device):
                rc = lib.lik_attention_backward(
                    ctypes.byref(a), out.data_ptr(), lse.data_ptr(), low.data_ptr(), g.data_ptr(),
                    0 if cu_q is not None else g.stride(0), g.stride(-3), g.stride(-2), _lib.ptr(gq), _lib.ptr(gk),
                    _lib.ptr(gv), _lib.ptr(ws), nbytes, _lib.stream_of(q))
            _lib.check(rc, "lik_attention_backward")
        return gq, gk if need_k else None, gv if need_v else None, None, None, None, None, None


def _check(q, k, v, causal, window, scale):
    """Shared argument checks; returns ``(left, right, scale)``."""
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"attention takes fp16 / bf16; got {q.dtype}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k and v must have one type; got {q.dtype}, {k.dtype}, {v.dtype}")
    if k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must be on the same device.")
    if k.shape != v.shape:
        raise ValueError(f"k and v must have one shape; got {tuple(k.shape)} and {tuple(v.shape)}")
    h, d, hk = q.shape[-2], q.shape[-1], k.shape[-2]
    if k.shape[-1] != d:
        raise ValueError(f"q and k must share the head dim; got {d} and {k.shape[-1]}")
    if not 1 <= d <= 128:
        raise ValueError(f"attention takes head dims of 1 to 128; got {d}")
    if h < 1 or hk < 1 or h % hk:
        raise ValueError(f"the heads of q ({h}) must be a multiple of those of k and v ({hk})")
    if window is not None and (not isinstance(window, int) or isinstance(window, bool) or window < 0):
        raise ValueError(f"window must be None or an int >= 0; got {window!r}")
    scale = d**-0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite; got {scale}")
    left = -1 if window is None else min(window, 2**30)
    return left, 0 if causal else left, scale


def _run(q, k, v, meta, qm, km, cu_q, cu_k):
    d = q.shape[-1]
    if _lib.differentiates(q, k, v):
        pad = -d % 8  # zero columns change no product; padded here so that autograd cuts the gradients
        if pad:
            q, k, v = (torch.nn.functional.pad(t, (0, pad)) for t in (q, k, v))
        out = _AttentionFn.apply(q, k, v, meta, qm, km, cu_q, cu_k)
    else:
        q, k, v = _lib.rows16(q, -3, _FAR), _lib.rows16(k, -3, _FAR), _lib.rows16(v, -3, _FAR)
        out, _, _ = _forward(q, k, v, meta, qm, km, cu_q, cu_k, False)
    return out[..., :d] if d % 8 else out


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    q_mask: torch.Tensor | None = None,
    k_mask: torch.Tensor | None = None,
    *,
    causal: bool = False,
    window: int | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention over padded sequences.

    Args:
        q: ``[n, Lq, H, d]`` fp16 / bf16, ``d`` at most 128 (a multiple of 8 in the
            kernels; other sizes are padded in a copy). Any strides (rows off 16 bytes, or
            tokens 2^24 elements apart, are copied).
        k, v: ``[n, Lk, Hk, d]``; ``H`` a multiple of ``Hk``.
        q_mask: ``[n, Lq]``, True = keep. Rows that it drops come out as zeros and
            give no gradient; whatever they hold is not used.
        k_mask: ``[n, Lk]``, True = keep. Either mask: lengths up to 2^18.
        causal: query i keeps the keys j <= i.
        window: query i keeps the keys with ``|i - j| <= window``.
        scale: of the scores (default ``d ** -0.5``), positive.

    Returns:
        ``[n, Lq, H, d]``; zeros for a query that keeps no key.
    """
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q, k and v must be [n, L, heads, d]; got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}. For packed inputs use `attention_varlen`.")
    if k.shape[0] != q.shape[0]:
        raise ValueError(f"q and k must have one batch size; got {q.shape[0]} and {k.shape[0]}")
    left, right, scale = _check(q, k, v, causal, window, scale)
    for name, m, x in (("q_mask", q_mask, q), ("k_mask", k_mask, k)):
        if m is None:
            continue
        if m.device != x.device:
            raise ValueError(f"{name} must be on the same device as {name[0]}; got {m.device} vs {x.device}.")
        if m.dim() != 2 or m.shape != x.shape[:2]:
            raise ValueError(f"{name} must be {list(x.shape[:2])}; got {tuple(m.shape)}")
        if x.shape[1] > 2**18:
            raise ValueError(f"{name} takes lengths up to {2**18}; got {x.shape[1]}")
    _lib.require_gpu(q)
    return _run(q, k, v, (left, right, scale, q.shape[1], k.shape[1]), _mask_i8(q_mask, q.shape[:2]),
                _mask_i8(k_mask, k.shape[:2]), None, None)


def attention_varlen(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor,
    max_seqlen_q: int | None = None,
    max_seqlen_k: int | None = None,
    *,
    causal: bool = False,
    window: int | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention over packed sequences.

    Args:
        q: ``[sum(Lq_i), H, d]`` fp16 / bf16; k, v: ``[sum(Lk_i), Hk, d]``.
        cu_seqlens_q, cu_seqlens_k: ``[n + 1]`` int32 cumulative offsets. Rows outside
            ``cu[0] .. cu[-1]`` are in no sequence: zeros, and no gradient.
        max_seqlen_q, max_seqlen_k: hard bounds on the lengths; inferred with one
            device->host sync each if omitted, otherwise checked by an on-device assert.
        causal, window, scale: as in :func:`attention`; positions count from each sequence's start.

    Returns:
        ``[sum(Lq_i), H, d]``.
    """
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"q, k and v must be packed [tokens, heads, d]; got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}. For padded inputs use `attention`.")
    left, right, scale = _check(q, k, v, causal, window, scale)
    for name, cu in (("cu_seqlens_q", cu_seqlens_q), ("cu_seqlens_k", cu_seqlens_k)):
        if cu.device != q.device:
            raise ValueError(f"{name} must be on the same device as q; got {cu.device} vs {q.device}.")
        if cu.dim() != 1 or cu.numel() < 1 or cu.is_floating_point():
            raise ValueError(f"{name} must be [n + 1] cumulative offsets; got {tuple(cu.shape)} {cu.dtype}")
    if cu_seqlens_q.numel() != cu_seqlens_k.numel():
        raise ValueError(f"cu_seqlens_q and cu_seqlens_k must name as many sequences; got "
                         f"{cu_seqlens_q.numel() - 1} and {cu_seqlens_k.numel() - 1}")
    _lib.require_gpu(q)
    cu_q = _i32(cu_seqlens_q)
    cu_k = cu_q if cu_seqlens_k is cu_seqlens_q else _i32(cu_seqlens_k)
    given = [(cu, None if m is None else int(m), name) for cu, m, name in (
        (cu_q, max_seqlen_q, "max_seqlen_q"), (cu_k, max_seqlen_k, "max_seqlen_k"))]
    if cu_k is cu_q and None not in (given[0][1], given[1][1]):  # one array: the tighter bound covers both
        assert_max_seqlens_cover(min(given, key=lambda g: g[1]))
    else:
        assert_max_seqlens_cover(*given)
    max_q, max_k = (seqlen_max(cu) if m is None else m for cu, m, _ in given)
    return _run(q, k, v, (left, right, scale, max_q, max_k), None, None, cu_q, cu_k)


__all__ = ["attention", "attention_varlen"]
