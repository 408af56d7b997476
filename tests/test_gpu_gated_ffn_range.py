"""gated_ffn of bf16 rows whose projections are far from 1: bf16 has fp32's range, so the gradients
keep their share of error at any size.

Bounds: as at size 1, two roundings to bf16 (of the gradients of both projections, and of the result), sqrt(2 / 3) u in the
2-norm when errors spread evenly, bounded by 1.25 u; what the backward pass reads of the forward's projections has to
carry next to no rounding of its own."""

import pytest
import torch

from encoder_plain import ROUNDOFF, gated_ffn64, off
from late_interaction_kernels.encoder import gated_ffn

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows,d,f", [(5, 64, 48), (64, 768, 1152), (300, 128, 200), (1030, 264, 520)])
@pytest.mark.parametrize("size", [1e-12, 1e-7, 1e-6, 1e-5, 1e-4, 1e-2, 1e3, 1e7, 1e15])
def test_gradients_of_projections_of_any_size(act, rows, d, f, size):
    print("[case]", act, rows, d, f, size, flush=True)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(rows, d, generator=g).to(BF)
    wi = (torch.randn(2 * f, d, generator=g) * d**-0.5 * size).to(BF)
    wo = (torch.randn(d, f, generator=g) * f**-0.5).to(BF)
    gy = torch.randn(rows, d, generator=g).to(BF)
    leaves = [t.double().requires_grad_() for t in (x, wi, wo)]
    y64 = gated_ffn64(*leaves, None, act)
    want = torch.autograd.grad(y64, leaves, gy.double())
    ts = [t.cuda().requires_grad_() for t in (x, wi, wo)]
    y = gated_ffn(*ts, activation=act)
    u = 1.25 * ROUNDOFF[BF]
    assert off(y, y64) <= u
    for name, a, b in zip(("x", "w_in", "w_out"), torch.autograd.grad(y, ts, gy.cuda()), want):
        assert off(a, b) <= u, name


def test_hidden_units_of_very_different_sizes():
    """Every unit by itself: tiny ones next to large ones keep their own gradients."""
    g = torch.Generator().manual_seed(4)
    rows, d, f = 200, 64, 64
    x = torch.randn(rows, d, generator=g).to(BF)
    size = torch.logspace(-9, 3, f)[torch.randperm(f, generator=g)]
    wi = (torch.randn(2, f, d, generator=g) * d**-0.5 * size[:, None]).to(BF).view(2 * f, d)
    wo = (torch.randn(d, f, generator=g) * f**-0.5).to(BF)
    gy = torch.randn(rows, d, generator=g).to(BF)
    leaves = [t.double().requires_grad_() for t in (x, wi, wo)]
    want = torch.autograd.grad(gated_ffn64(*leaves, None, "silu"), leaves, gy.double())
    ts = [t.cuda().requires_grad_() for t in (x, wi, wo)]
    got = torch.autograd.grad(gated_ffn(*ts, activation="silu"), ts, gy.cuda())
    for i in range(2 * f):  # 64 values a row: their errors' 2-norm, at most u each for both roundings
        assert off(got[1][i], want[1][i]) <= 1.25 * ROUNDOFF[BF], i


def test_values_that_are_not_finite_stay_in_their_rows():
    g = torch.Generator().manual_seed(6)
    x = torch.randn(70, 64, generator=g).to(BF)
    wi, wo = torch.randn(128, 64, generator=g).to(BF), torch.randn(64, 64, generator=g).to(BF)
    gy = torch.randn(70, 64, generator=g).to(BF).cuda()

    def grad(x):
        xs = x.cuda().requires_grad_()
        return torch.autograd.grad(gated_ffn(xs, wi.cuda(), wo.cuda()), xs, gy)[0]

    want = grad(x)
    x[3, 1], x[40, 2] = float("nan"), float("inf")
    got = grad(x)
    rest = [i for i in range(70) if i not in (3, 40)]
    assert torch.equal(got[rest], want[rest]) and torch.isnan(got[3]).all() and not torch.isfinite(got[40]).any()
