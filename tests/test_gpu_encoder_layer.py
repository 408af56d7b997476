"""The encoder operators together: a layer against plain 64-bit operators, and the training example."""

import importlib.util
from pathlib import Path

import pytest
import torch

from encoder_plain import ROUNDOFF, attention64, gated_ffn64, keep_pairs, layer_norm64, off

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "train_encoder.py"
    spec = importlib.util.spec_from_file_location("train_encoder", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("window", [None, 7])
def test_layer_and_its_gradients(window):
    """About a dozen roundings to bf16 lie between the layer's input and its output (and as many
    back): independent ones of u / sqrt(3) each add up to 2 u, bounded by 4 u."""
    m = _example()
    torch.manual_seed(1)
    n, length, d, h, hk, f = 3, 50, 128, 4, 2, 192
    layer = m.EncoderLayer(d, h, hk, f, window).cuda().to(torch.bfloat16)
    mask = torch.arange(length)[None] < torch.tensor([50, 17, 33])[:, None]
    x, s, gy = (torch.randn(n, length, d).to(torch.bfloat16) for _ in range(3))
    gy = gy * mask[..., None]
    xs, ss = x.cuda().requires_grad_(), s.cuda().requires_grad_()
    y, t = layer(xs, ss, mask.cuda())
    names = ["w_qkv", "w_att", "w_in", "w_out"]
    got = torch.autograd.grad((y + t), [xs, ss] + [getattr(layer, k) for k in names], gy.cuda())

    p = {k: v.detach().cpu().double().requires_grad_() for k, v in layer.named_parameters()}
    x64, s64 = x.double().requires_grad_(), s.double().requires_grad_()
    y64, t64 = layer_norm64(x64, p["norm_att"], None, s64, 1e-5, None)
    qkv = (y64 @ p["w_qkv"].t()).view(n, length, h + 2 * hk, d // h)
    q, k, v = qkv.split([h, hk, hk], 2)
    keep = keep_pairs(length, length, False, window)
    a = torch.stack([attention64(q[i], k[i], v[i], keep & mask[i][None] & mask[i][:, None], (d // h) ** -0.5)
                     for i in range(n)])
    y64, t64 = layer_norm64(a.reshape(n, length, -1) @ p["w_att"].t(), p["norm_ffn"], None, t64, 1e-5, None)
    out = gated_ffn64(y64.reshape(-1, d), p["w_in"], p["w_out"], None, "gelu").view(n, length, d) + t64
    want = torch.autograd.grad(out, [x64, s64] + [p[k] for k in names], gy.double())
    u = 4 * ROUNDOFF[torch.bfloat16]
    assert off((y.double() + t.double()).cpu()[mask], out[mask]) <= u
    for name, a, b in zip(["x", "s"] + names, got, want):
        assert off(a, b) <= u, name


def test_training_example_learns():
    losses = _example().train(steps=30)
    assert all(map(lambda x: x == x, losses))
    assert sum(losses[-5:]) / 5 < 0.6 * sum(losses[:5]) / 5, losses
