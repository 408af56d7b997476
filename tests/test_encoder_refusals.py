"""What the encoder operators refuse, before any launch (no GPU needed)."""

import pytest
import torch

from late_interaction_kernels.encoder import attention, attention_varlen, gated_ffn, layer_norm

BF = torch.bfloat16


def _z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def test_layer_norm_refusals():
    x, w = _z(4, 16), _z(16)
    for bad, err in (((_z(4, 16, dtype=torch.float64), w), TypeError), ((x, _z(15)), ValueError),
                     ((x, _z(16, dtype=torch.float16)), TypeError), ((x, w, _z(16, dtype=torch.float32)), ValueError),
                     ((x, w, None, _z(4, 15)), ValueError), ((x, w, None, _z(4, 16, dtype=torch.float32)), ValueError),
                     ((_z(2, 8193), _z(8193)), ValueError), ((_z(4, 0), _z(0)), ValueError)):
        with pytest.raises(err):
            layer_norm(*bad)
    with pytest.raises(RuntimeError, match="GPU"):
        layer_norm(x, w)


def test_gated_ffn_refusals():
    x, wi, wo = _z(4, 16), _z(48, 16), _z(16, 24)
    for bad, err in (((x.float(), wi.float(), wo.float()), TypeError), ((x, wi.half(), wo), TypeError),
                     ((x, _z(47, 16), wo), ValueError), ((x, wi, _z(15, 24)), ValueError),
                     ((x, wi, _z(16)), ValueError), ((x, wi, wo, _z(4, 15)), ValueError),
                     ((x, wi, wo, x.float()), ValueError)):
        with pytest.raises(err):
            gated_ffn(*bad)
    with pytest.raises(ValueError, match="activation"):
        gated_ffn(x, wi, wo, activation="relu")
    with pytest.raises(RuntimeError, match="GPU"):
        gated_ffn(x, wi, wo)


def test_attention_refusals():
    q, k = _z(2, 5, 4, 16), _z(2, 7, 2, 16)
    for bad, err in (((q.float(), k.float(), k.float()), TypeError), ((q, k.half(), k), TypeError),
                     ((q[0], k, k), ValueError), ((q, k, k[:, :6]), ValueError), ((q, k[:1], k[:1]), ValueError),
                     ((q, _z(2, 7, 3, 16), _z(2, 7, 3, 16)), ValueError), ((q, _z(2, 7, 2, 8), _z(2, 7, 2, 8)), ValueError),
                     ((_z(1, 2, 2, 136),) * 3, ValueError), ((q, k, k, _z(2, 6).bool()), ValueError),
                     ((q, k, k, None, _z(2, 6).bool()), ValueError), ((q, k, k, None, _z(7).bool()), ValueError)):
        with pytest.raises(err):
            attention(*bad)
    for kw in ({"window": -1}, {"window": 2.0}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("inf")}):
        with pytest.raises(ValueError):
            attention(q, k, k, **kw)
    with pytest.raises(RuntimeError, match="GPU"):
        attention(q, k, k)


def test_attention_varlen_refusals():
    q, cu = _z(9, 2, 16), torch.tensor([0, 4, 9], dtype=torch.int32)
    for bad in ((q[None], q, q, cu, cu), (q, q, q, cu.float(), cu), (q, q, q, cu, cu[:2]), (q, q, q, cu[None], cu)):
        with pytest.raises(ValueError):
            attention_varlen(*bad)
    with pytest.raises(RuntimeError, match="GPU"):
        attention_varlen(q, q, q, cu, cu)
