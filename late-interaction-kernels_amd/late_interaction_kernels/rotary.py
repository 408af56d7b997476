"""``rotary``: rotary positions of queries and keys, padded, packed or at given
positions, differentiable; ``rotary_frequencies``: the frequencies it takes.

Pair i of a head is turned by ``position * frequencies[i]``. The angle is computed
and reduced in 64 bits (far positions keep their phase), the rotation is fp32 and
rounded once. The gradient is the rotation the other way; being linear it can be
differentiated again.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from ._core import _i32

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_LARGEST = torch.finfo(torch.float32).max


def rotary_frequencies(
    dim: int,
    base: float = 10000.0,
    *,
    scaling: str | None = None,
    factor: float = 1.0,
    original_length: int | None = None,
    low: float | None = None,
    high: float | None = None,
    device: torch.device | str | None = None,
) -> tuple[torch.Tensor, float]:
    """Frequencies of ``dim`` rotated elements and the amplitude that goes with them.

    ``f_i = base ** (-2 i / dim)``, in radians a position, ``i < dim / 2``. ``scaling``
    adapts them to contexts ``factor`` times as long as the ``original_length`` a model was trained on:

    - ``"linear"``: ``f_i / factor``.
    - ``"ntk"``: the base times ``factor ** (dim / (dim - 2))``, so that the lowest frequency
      is divided by ``factor`` and the highest is kept.
    - ``"bands"``: by the turns ``original_length * f_i / (2 pi)`` of a pair over the original
      length: at most ``low`` (default 1) turns ``f_i / factor``, at least ``high`` (default 4) ``f_i``, between
      them a blend that is linear in the turns.
    - ``"yarn"`` (Peng et al., "YaRN: Efficient context window extension of large language
      models", 2023): the blend is linear in the pair's index, between the pairs that turn
      ``high`` (default 32, rounded down) and ``low`` (default 1, rounded up) times; the amplitude is
      ``0.1 ln factor + 1``. As in the models that were trained so, and not in the paper, the last of them is at
      most pair ``dim - 1``, and where both are one pair the blend takes 0.001 of an index.

    Returns:
        ``(frequencies, amplitude)``: fp64 ``[dim / 2]`` on ``device``, and 1.0 except for "yarn".
    """
    if dim < 2 or dim % 2:
        raise ValueError(f"dim must be even and at least 2; got {dim}")
    if not (base > 0 and math.isfinite(base)):
        raise ValueError(f"base must be positive and finite; got {base}")
    if not (factor >= 1 and math.isfinite(factor)):
        raise ValueError(f"factor must be finite and at least 1; got {factor}")
    if scaling not in (None, "linear", "ntk", "bands", "yarn"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk', 'bands' or 'yarn'; got {scaling!r}")
    if scaling is None and factor != 1:
        raise ValueError("factor needs a scaling")
    i = torch.arange(dim // 2, dtype=torch.float64)
    amplitude = 1.0
    if scaling == "ntk":
        if dim < 4:
            raise ValueError("'ntk' needs a dim of at least 4")
        base = base * factor ** (dim / (dim - 2))
    f = base ** (-2.0 * i / dim)
    if scaling == "linear":
        f = f / factor
    elif scaling in ("bands", "yarn"):
        if original_length is None or original_length < 1:
            raise ValueError(f"{scaling!r} needs the original_length; got {original_length}")
        low = 1.0 if low is None else float(low)
        high = (4.0 if scaling == "bands" else 32.0) if high is None else float(high)
        if not 0 < low < high:
            raise ValueError(f"low and high must be 0 < low < high; got {low} and {high}")
        if scaling == "bands":
            keep = ((original_length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        else:
            if base <= 1:
                raise ValueError(f"'yarn' needs a base above 1; got {base}")

            def pair(turns):  # the (fractional) pair that turns so many times over the original length
                return dim * math.log(original_length / (2 * math.pi * turns)) / (2 * math.log(base))

            first, last = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), dim - 1)
            keep = 1 - ((i - first) / max(last - first, 0.001)).clamp(0, 1)
            amplitude = 0.1 * math.log(factor) + 1
        f = f * keep + f / factor * (1 - keep)
    return f.to(device), amplitude


def _launch(q, k, frequencies, positions, cu, meta):
    """``(q', k')`` of the tensors that are not None."""
    offset, interleaved, amplitude, inverse = meta
    x = k if q is None else q
    *lead, _, d = x.shape
    outq = outk = None
    hq = hk = qp = kp = qn = ql = qh = kn = kl = kh = pn = pl = pos = bits = 0
    some = False
    if q is not None:
        outq = torch.empty_like(q, memory_format=torch.contiguous_format)
        hq, qp, some = q.size(-2), q.data_ptr(), q.numel() != 0
        *outer, ql, qh, _ = q.stride()
        if outer:
            qn = outer[0]
    if k is not None:
        outk = torch.empty_like(k, memory_format=torch.contiguous_format)
        hk, kp, some = k.size(-2), k.data_ptr(), some or k.numel() != 0
        *outer, kl, kh, _ = k.stride()
        if outer:
            kn = outer[0]
    if not some:
        return outq, outk
    if len(lead) == 1:
        n, length = 1 if cu is None else cu.numel() - 1, lead[0]
    else:
        n, length = lead
    if positions is not None:
        pos, bits = positions.data_ptr(), 8 * positions.element_size()
        *outer, pl = positions.stride()
        if outer:
            pn = outer[0]
    a = _lib.pack_rotary(qp, kp, _lib.DTYPE_CODE[x.dtype], hq, hk, d, n, length, qn, ql, qh, kn, kl, kh,
                         0 if cu is None else cu.data_ptr(), pos, pn, pl, offset, frequencies.data_ptr(), bits,
                         8 * frequencies.element_size(), frequencies.numel(), interleaved, inverse, amplitude)
    with _lib.on_device(x.device):
        rc = _lib.load().lik_rotary(a, _lib.ptr(outq), _lib.ptr(outk), _lib.stream_of(x))
    _lib.check(rc, "lik_rotary")
    return outq, outk


def _unit(t):
    """``t`` with a contiguous last dim."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, frequencies, positions, cu, meta):
        ctx.save_for_backward(frequencies, positions, cu)
        ctx.meta = meta
        ctx.set_materialize_grads(False)
        return _launch(_unit(q), _unit(k), frequencies, positions, cu, meta)

    @staticmethod
    def backward(ctx, gq, gk):
        offset, interleaved, amplitude, inverse = ctx.meta
        need_q, need_k, *_ = ctx.needs_input_grad
        gq, gk = gq if need_q else None, gk if need_k else None
        if gq is not None or gk is not None:
            meta = (offset, interleaved, amplitude, not inverse)
            if torch.is_grad_enabled():
                gq, gk = _RotaryFn.apply(gq, gk, *ctx.saved_tensors, meta)
            else:
                gq, gk = _launch(_unit(gq), _unit(gk), *ctx.saved_tensors, meta)
        return gq, gk, None, None, None, None


def rotary(
    q: torch.Tensor,
    k: torch.Tensor | None = None,
    *,
    frequencies: torch.Tensor,
    positions: torch.Tensor | None = None,
    cu_seqlens: torch.Tensor | None = None,
    offset: int = 0,
    interleaved: bool = False,
    amplitude: float = 1.0,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Rotary positions of ``q`` and (in the same launch) ``k``, in front of :func:`attention.attention`.

    Args:
        q: ``[n, L, H, d]`` or packed ``[T, H, d]``, fp16 / bf16 / fp32, ``d`` at most 1024, any strides.
        k: the same with heads of its own number, or None.
        frequencies: ``[r / 2]`` fp32 / fp64, radians a position (:func:`rotary_frequencies`);
            the first ``r`` elements of each head are turned, the others are copied.
        positions: int32 / int64 ``[n, L]`` or ``[L]`` (packed: ``[T]``); None counts from
            ``offset`` at the start of each sequence.
        cu_seqlens: ``[s + 1]`` int32 cumulative offsets of packed sequences, where positions are
            counted. Rows outside ``cu[0] .. cu[-1]`` come out as zeros and get no gradient.
        interleaved: pairs are elements ``(2 i, 2 i + 1)`` instead of ``(i, i + r / 2)``.
        amplitude: of the turned elements.

    Returns:
        ``q'`` of the shape and type of ``q``, or ``(q', k')``; contiguous.
    """
    shape, dtype, device = q.shape, q.dtype, q.device
    if len(shape) not in (3, 4):
        raise ValueError(f"q must be [n, L, heads, d] or packed [tokens, heads, d]; got {tuple(shape)}")
    if dtype not in _DTYPES:
        raise TypeError(f"rotary takes fp16 / bf16 / fp32; got {dtype}")
    *lead, heads, d = shape
    if k is not None:
        *k_lead, k_heads, k_d = k.shape
        if k.dtype != dtype:
            raise TypeError(f"q and k must have one type; got {dtype} and {k.dtype}")
        if k_lead != lead or k_d != d:
            raise ValueError(f"k must match q ({tuple(shape)}) but in its heads; got {tuple(k.shape)}")
        if k_heads > 65536:
            raise ValueError("rotary takes at most 65536 heads")
        if k.device != device:
            raise ValueError("q, k, frequencies, positions and cu_seqlens must be on the same device.")
    if heads > 65536:
        raise ValueError("rotary takes at most 65536 heads")
    if not 2 <= d <= 1024:
        raise ValueError(f"rotary takes head dims of 2 to 1024; got {d}")
    if frequencies.dim() != 1 or not 1 <= frequencies.numel() <= d // 2:
        raise ValueError(f"frequencies must be [r / 2] with 2 <= r <= {d}; got {tuple(frequencies.shape)}")
    if frequencies.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"frequencies must be fp32 or fp64; got {frequencies.dtype}")
    if frequencies.requires_grad:
        if torch.is_grad_enabled():
            raise ValueError("rotary gives no gradient to its frequencies; pass frequencies.detach()")
        frequencies = frequencies.detach()
    if not isinstance(offset, int) or isinstance(offset, bool) or abs(offset) > 2**31:
        raise ValueError(f"offset must be an int of at most 2^31; got {offset!r}")
    if positions is not None:
        if cu_seqlens is not None or offset != 0:
            raise ValueError("positions say everything: give them without cu_seqlens and offset")
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"positions must be int32 or int64; got {positions.dtype}")
        if list(positions.shape) not in (lead, lead[1:] or lead):
            raise ValueError(f"positions must be {lead}{' or [L]' if len(lead) == 2 else ''}; got "
                             f"{tuple(positions.shape)}")
        if positions.device != device:
            raise ValueError("q, k, frequencies, positions and cu_seqlens must be on the same device.")
    elif cu_seqlens is not None:
        if len(lead) != 1:
            raise ValueError("cu_seqlens go with packed [tokens, heads, d]")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"cu_seqlens must be [s + 1] cumulative offsets; got {tuple(cu_seqlens.shape)} "
                             f"{cu_seqlens.dtype}")
        if cu_seqlens.device != device:
            raise ValueError("q, k, frequencies, positions and cu_seqlens must be on the same device.")
    elif len(lead) == 1:
        raise ValueError("packed rows need cu_seqlens or positions")
    amplitude = float(amplitude)
    if not abs(amplitude) <= _LARGEST:
        raise ValueError(f"amplitude must be a finite fp32 number; got {amplitude}")
    if frequencies.device != device:
        raise ValueError("q, k, frequencies, positions and cu_seqlens must be on the same device.")
    _lib.require_gpu(q)
    if not frequencies.is_contiguous():
        frequencies = frequencies.contiguous()
    meta = (offset, bool(interleaved), amplitude, False)
    cu = _i32(cu_seqlens)
    if _lib.differentiates(q, k):
        out = _RotaryFn.apply(q, k, frequencies, positions, cu, meta)
    else:
        out = _launch(_unit(q), _unit(k), frequencies, positions, cu, meta)
    return out[0] if k is None else out


__all__ = ["rotary", "rotary_frequencies"]
