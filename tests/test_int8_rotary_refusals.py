"""What the rotation, the 8-bit tokens and the linear layer on them refuse, before any launch (no GPU needed)."""

import math

import pytest
import torch

from late_interaction_kernels.encoder import (dequantize_int8_per_token, linear_int8, quantize_int8_per_token, rotary,
                                              rotary_frequencies)

BF, I8 = torch.bfloat16, torch.int8


def _z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def test_rotary_refusals():
    q, k, f = _z(2, 5, 4, 16), _z(2, 5, 2, 16), _z(8, dtype=torch.float64)
    p, cu = _z(9, 2, 16), torch.tensor([0, 4, 9], dtype=torch.int32)
    pos = torch.zeros(2, 5, dtype=torch.int64)
    for args, kw, err in (
            ((q.double(),), {}, TypeError), ((q, k.half()), {}, TypeError), ((q[0, 0],), {}, ValueError),
            ((q, k[:1]), {}, ValueError), ((q, k[..., :8]), {}, ValueError), ((q, k[0]), {}, ValueError),
            ((q,), {"frequencies": f[:0]}, ValueError), ((q,), {"frequencies": _z(9, dtype=torch.float32)}, ValueError),
            ((q,), {"frequencies": f[None]}, ValueError), ((q,), {"frequencies": f.to(BF)}, TypeError),
            ((q,), {"frequencies": f.clone().requires_grad_()}, ValueError),
            ((q,), {"positions": pos.float()}, TypeError), ((q,), {"positions": pos[:, :4]}, ValueError),
            ((q,), {"positions": pos[0, :2]}, ValueError), ((q,), {"positions": pos, "offset": 1}, ValueError),
            ((q,), {"cu_seqlens": cu}, ValueError), ((p,), {}, ValueError),
            ((p,), {"cu_seqlens": cu, "positions": pos[0]}, ValueError), ((p,), {"cu_seqlens": cu.float()}, ValueError),
            ((p,), {"cu_seqlens": cu[None]}, ValueError), ((p,), {"cu_seqlens": cu[:0]}, ValueError),
            ((q,), {"offset": 1.0}, ValueError), ((q,), {"offset": 2**40}, ValueError),
            ((q,), {"amplitude": float("nan")}, ValueError), ((_z(1, 2, 2, 1026),), {}, ValueError),
            ((_z(1, 2, 2, 1),), {"frequencies": f[:1]}, ValueError)):
        with pytest.raises(err):
            rotary(*args, **{"frequencies": f, **kw})
    for kw in ({}, {"positions": pos}, {"positions": pos[0].int()}, {"offset": -3}):
        with pytest.raises(RuntimeError, match="GPU"):
            rotary(q, k, frequencies=f, **kw)
    with pytest.raises(RuntimeError, match="GPU"):
        rotary(p, frequencies=f, cu_seqlens=cu)


def test_rotary_frequencies():
    f, amp = rotary_frequencies(8)
    assert f.dtype == torch.float64 and amp == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001]).double())
    assert torch.equal(rotary_frequencies(8, scaling="linear", factor=4.0)[0], f / 4)
    g, _ = rotary_frequencies(8, scaling="ntk", factor=4.0)
    assert abs(float(g[0]) - 1) < 1e-12 and abs(float(g[-1] / f[-1]) - 0.25) < 1e-12
    for scaling in ("bands", "yarn"):
        same, one = rotary_frequencies(64, scaling=scaling, factor=1.0, original_length=2048)
        assert torch.allclose(same, rotary_frequencies(64)[0]) and one == 1.0
        g, amp = rotary_frequencies(64, scaling=scaling, factor=8.0, original_length=2048)
        ratio = g / rotary_frequencies(64)[0]
        assert abs(float(ratio[0]) - 1) < 1e-12 and abs(float(ratio[-1]) - 0.125) < 1e-12
        assert bool((ratio.diff() <= 1e-12).all())  # slower pairs are stretched more
        assert amp == (1.0 if scaling == "bands" else 0.1 * math.log(8) + 1)
    turns = 2048 * rotary_frequencies(64)[0] / (2 * math.pi)
    ratio = rotary_frequencies(64, scaling="bands", factor=8.0, original_length=2048)[0] / rotary_frequencies(64)[0]
    assert torch.allclose(ratio[turns >= 4], torch.ones(()).double())
    assert torch.allclose(ratio[turns <= 1], torch.full((), 0.125).double())
    for bad in ({"dim": 7}, {"dim": 0}, {"dim": 8, "base": 0.0}, {"dim": 8, "factor": 2.0}, {"dim": 8, "scaling": "x"},
                {"dim": 8, "scaling": "linear", "factor": 0.5}, {"dim": 8, "scaling": "yarn", "factor": 2.0},
                {"dim": 2, "scaling": "ntk", "factor": 2.0}, {"dim": 8, "scaling": "bands", "original_length": 0},
                {"dim": 8, "scaling": "bands", "original_length": 64, "low": 4.0, "high": 4.0}):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_int8_token_refusals():
    for bad, err in ((_z(4, 8, dtype=torch.float64), TypeError), (_z(4, 8, dtype=I8), TypeError), (_z(4, 0), ValueError),
                     (torch.tensor(1.0), ValueError)):
        with pytest.raises(err):
            quantize_int8_per_token(bad)
    q, s = _z(4, 8, dtype=I8), _z(4, dtype=torch.float32)
    for args, err in (((q.float(), s), TypeError), ((q, s.half()), TypeError), ((q, s[:3]), ValueError),
                      ((q, s[:, None]), ValueError), ((q, s, torch.float64), TypeError), ((q[:, :0], s), ValueError)):
        with pytest.raises(err):
            dequantize_int8_per_token(*args)
    with pytest.raises(RuntimeError, match="GPU"):
        quantize_int8_per_token(_z(4, 8))
    with pytest.raises(RuntimeError, match="GPU"):
        dequantize_int8_per_token(q, s)


def test_linear_int8_refusals():
    x, w, ws = _z(4, 16), _z(10, 16, dtype=I8), _z(10, dtype=torch.float32)
    xq, xs = _z(4, 16, dtype=I8), _z(4, dtype=torch.float32)
    for args, kw, err in (
            ((x.double(), w, ws), {}, TypeError), ((x, w.float(), ws), {}, TypeError), ((x, w, ws.half()), {}, TypeError),
            ((x, w[:, :15], ws), {}, ValueError), ((x, w[0], ws), {}, ValueError), ((x, w, ws[:9]), {}, ValueError),
            ((x, w, ws), {"x_scale": xs}, ValueError), ((xq, w, ws), {}, ValueError),
            ((xq, w, ws), {"x_scale": xs[:3]}, ValueError), ((xq, w, ws), {"x_scale": xs.half()}, ValueError),
            ((x, w, ws), {"activation": "relu"}, ValueError), ((x, w[:9], ws[:9]), {"gated": True}, ValueError),
            ((x, w, ws, _z(9)), {}, ValueError), ((x, w, ws, _z(10, dtype=torch.float16)), {}, ValueError),
            ((x, w, ws, None, _z(4, 9)), {}, ValueError), ((x, w, ws, None, _z(4, 10).float()), {}, ValueError),
            ((x, w, ws, None, _z(4, 10)), {"gated": True}, ValueError), ((x, w, ws), {"out_dtype": I8}, TypeError),
            ((_z(1, 131072), _z(1, 131072, dtype=I8), ws[:1]), {}, ValueError), ((x, w[:0], ws[:0]), {}, ValueError)):
        with pytest.raises(err):
            linear_int8(*args, **kw)
    with pytest.raises(RuntimeError, match="GPU"):
        linear_int8(x, w, ws)
    with pytest.raises(RuntimeError, match="GPU"):
        linear_int8(xq, w, ws, x_scale=xs, gated=True, activation="gelu", out_dtype=torch.float32)
