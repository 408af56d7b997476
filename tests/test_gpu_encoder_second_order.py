"""Gradients of gradients: the encoder operators have none and say so, instead of
taking their first gradients for constants."""

import pytest
import torch

from late_interaction_kernels import encoder

pytestmark = pytest.mark.gpu


def _attention(x):
    y = x.view(2, 6, 2, 16)
    return encoder.attention(y, y, y)


def _attention_padded_heads(x):
    y = x.view(2, 6, 4, 8)[..., :5]
    return encoder.attention(y, y, y)


def _layer_norm(x):
    w = torch.ones(32, device="cuda")
    y, total = encoder.layer_norm(x, w, None, x)
    return y + total


def _gated_ffn(x):
    w = torch.full((32, 32), 0.1, dtype=x.dtype, device="cuda")
    return encoder.gated_ffn(x, torch.cat([w, w]), w, x)


@pytest.mark.parametrize("op", [_attention, _attention_padded_heads, _layer_norm, _gated_ffn])
def test_second_gradients_are_refused(op):
    x = torch.randn(12, 32, generator=torch.Generator().manual_seed(3)).to("cuda", torch.bfloat16).requires_grad_()
    out = op(x).float().square().sum()
    (first,) = torch.autograd.grad(out, x, create_graph=True)
    (plain,) = torch.autograd.grad(op(x).float().square().sum(), x)
    assert torch.equal(first.detach(), plain)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first.float().square().sum().backward()
