"""Forward-mode derivatives: the encoder operators have none and say so, instead of dropping the
tangents of their inputs."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from late_interaction_kernels import encoder

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _attention(x):
    return encoder.attention(x.view(2, 6, 2, 16), *(torch.ones(2, 6, 2, 16, dtype=BF, device="cuda") for _ in range(2)))


def _attention_values(x):
    ones = torch.ones(2, 6, 2, 16, dtype=BF, device="cuda")
    return encoder.attention(ones, ones, x.view(2, 6, 2, 16))


def _varlen(x):
    cu = torch.tensor([0, 5, 12], dtype=torch.int32, device="cuda")
    ones = torch.ones(12, 2, 16, dtype=BF, device="cuda")
    return encoder.attention_varlen(ones, x.view(12, 2, 16), ones, cu, cu, 7, 7)


def _layer_norm(x):
    return encoder.layer_norm(x, torch.ones(32, device="cuda"))


def _layer_norm_residual(x):
    return encoder.layer_norm(torch.ones(12, 32, dtype=BF, device="cuda"), torch.ones(32, device="cuda"), None, x)


def _gated_ffn(x):
    w = torch.full((32, 32), 0.1, dtype=BF, device="cuda")
    return encoder.gated_ffn(x, torch.cat([w, w]), w)


def _gated_ffn_weight(x):
    w = torch.full((32, 32), 0.1, dtype=BF, device="cuda")
    return encoder.gated_ffn(torch.ones(5, 32, dtype=BF, device="cuda"), torch.cat([w, w]), x[:12].repeat(3, 1)[:32])


@pytest.mark.parametrize("op", [_attention, _attention_values, _varlen, _layer_norm, _layer_norm_residual, _gated_ffn,
                                _gated_ffn_weight])
def test_tangents_are_refused(op):
    x = torch.randn(12, 32, device="cuda").to(BF)
    want = op(x)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="jvp"):
            op(fwd.make_dual(x, torch.ones_like(x)))
        with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp"):
            op(fwd.make_dual(x, torch.ones_like(x)))
        got = op(x)  # without a tangent: as outside
    for a, b in zip(*((t if isinstance(t, tuple) else (t,)) for t in (got, want))):
        assert torch.equal(a, b)
