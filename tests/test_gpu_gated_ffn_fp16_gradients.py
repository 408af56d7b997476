"""gated_ffn of fp16 rows: gradients of any size. What lies between the products may leave fp16's range (largest
value 65504, spacing 2^-24 at the lower end) although neither the inputs nor the results do.

Bounds: two roundings, 1.25 u of the result's 2-norm as at size 1, and half a spacing of 2^-24 an element for the rounding of the
result itself."""

import pytest
import torch

from encoder_plain import ROUNDOFF, gated_ffn64
from late_interaction_kernels.encoder import gated_ffn

pytestmark = pytest.mark.gpu
FP = torch.float16


def _check(name, got, want):
    assert torch.isfinite(got).all(), name
    err = float((got.double().cpu() - want).norm())
    assert err <= 1.25 * ROUNDOFF[FP] * float(want.norm()) + 2.0**-25 * want.numel() ** 0.5, name


def _make(rows, d, f, sx, si, so, sg):
    g = torch.Generator().manual_seed(8)
    return tuple(t.to(FP) for t in (torch.randn(rows, d, generator=g) * sx, torch.randn(2 * f, d, generator=g) * d**-0.5 * si,
                                    torch.randn(d, f, generator=g) * f**-0.5 * so, torch.randn(rows, d, generator=g) * sg))


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("rows,d,f", [(40, 64, 48), (64, 768, 1152), (1024, 256, 384), (1500, 264, 520)])
@pytest.mark.parametrize("size", [1e-6, 1e-5, 1e-4, 1e-2, 1.0, 100.0])
def test_small_and_large_gradients(act, rows, d, f, size):
    print("[case]", act, rows, d, f, size, flush=True)
    x, wi, wo, gy = _make(rows, d, f, 1.0, 1.0, 1.0, size)
    leaves = [t.double().requires_grad_() for t in (x, wi, wo)]
    want = torch.autograd.grad(gated_ffn64(*leaves, None, act), leaves, gy.double())
    ts = [t.cuda().requires_grad_() for t in (x, wi, wo)]
    for name, a, b in zip(("x", "w_in", "w_out"), torch.autograd.grad(gated_ffn(*ts, activation=act), ts, gy.cuda()), want):
        _check(name, a, b)


@pytest.mark.parametrize("sx,si,so,sg", [(256.0, 2.0**-4, 1.0, 2000.0), (1.0, 2.0**-7, 1.0, 1e-3), (1.0, 1.0, 2.0**-8, 1e-3)])
def test_weights_of_other_sizes(sx, si, so, sg):
    """Large gradients over large inputs pass 65504 between the products; small weights push them under 2^-14."""
    print("[case]", sx, si, so, sg, flush=True)
    x, wi, wo, gy = _make(500, 128, 192, sx, si, so, sg)
    leaves = [t.double().requires_grad_() for t in (x, wi)]
    want = torch.autograd.grad(gated_ffn64(*leaves, wo.double(), None, "silu"), leaves, gy.double())
    ts = [t.cuda().requires_grad_() for t in (x, wi)]
    got = torch.autograd.grad(gated_ffn(*ts, wo.cuda(), activation="silu"), ts, gy.cuda())
    _check("x", got[0], want[0])
    if sx == 1:  # (else w_in's gradient is past fp16)
        _check("w_in", got[1], want[1])


def test_one_large_row():
    """A row whose gradient is 4096 times the others': theirs stay as exact."""
    x, wi, wo, gy = _make(600, 128, 192, 1.0, 1.0, 1.0, 2.0**-9)
    gy[77] *= 4096
    x64 = x.double().requires_grad_()
    (want,) = torch.autograd.grad(gated_ffn64(x64, wi.double(), wo.double(), None, "gelu"), x64, gy.double())
    xs = x.cuda().requires_grad_()
    (got,) = torch.autograd.grad(gated_ffn(xs, wi.cuda(), wo.cuda()), xs, gy.cuda())
    rest = torch.arange(600) != 77
    _check("others", got[rest.cuda()], want[rest])
    _check("large", got[77], want[77])


def test_gradients_that_are_zero_or_not_finite():
    x, wi, wo, gy = _make(100, 64, 96, 1.0, 1.0, 1.0, 1.0)
    ts = [t.cuda().requires_grad_() for t in (x, wi, wo)]
    y = gated_ffn(*ts)
    for t in torch.autograd.grad(y, ts, torch.zeros_like(y), retain_graph=True):
        assert not t.any()
    (want,) = torch.autograd.grad(y, ts[:1], gy.cuda(), retain_graph=True)
    for bad in (float("nan"), float("inf")):
        g2 = gy.clone()
        g2[7] = bad
        (got,) = torch.autograd.grad(y, ts[:1], g2.cuda(), retain_graph=True)
        rest = torch.arange(100, device="cuda") != 7
        _check("rest", got[rest], want[rest].double().cpu())
        assert not torch.isfinite(got[7]).any()
