"""Activations of ``linear_int8`` with fp32 outputs. The sums are zeros, so the bias alone goes in, exactly.

Bounds, in units of 2^-24 of the result (a rounding is off by 1, the hardware's exponential by 2):
gelu: 3 x^2 / 2 from the exponent's three roundings (of log2 e / 2 and two products), 2 from the exponential, 1 from the reciprocal and
1 from its argument, 1 for the polynomial's fit, 1 from the rest of its sum's roundings (shares of the value), 1 for each of the last
three products or sums, of which a positive x sees only its tail's share: 3 x^2 / 2 + 9.
silu: 4 from the exponential, 1 from the sum, 1 from the reciprocal, 2 products: 8. gelu_tanh: its exponent w has six roundings (of 0.0447, z^2,
the cubic term's sum, of sqrt(8 / pi), two products), each worth w (1 - sigmoid(w)), and 8 more as silu. An exponential under 2^-126 is
zero, which takes up to 88 * 2^-126 < 2^-119 off these two."""

import math

import pytest
import torch

from late_interaction_kernels.encoder import linear_int8

pytestmark = pytest.mark.gpu
FP, I8 = torch.float32, torch.int8
# few rows; tiles of 128 x 64 (gated: 64 x 128), 256 x 128, and walked ones of 256 x 256 and 256 x 192
SIZES = [(3, 4096), (70, 2050), (16481, 513), (66001, 256), (66001, 192)]


def _want(v, act):
    v = v.double()
    if act == "gelu":
        a = v * 0.5 * torch.special.erfc(-v / math.sqrt(2))
        return a, a.abs() * (1.5 * v * v + 9) * 2.0**-24 + 2.0**-146
    if act == "silu":
        a = v * torch.sigmoid(v)
        return a, a.abs() * 2.0**-21 + 2.0**-119
    w = math.sqrt(8 / math.pi) * (v + 0.044715 * v**3)
    a = v * torch.sigmoid(w)
    return a, a.abs() * (6 * w.abs() * torch.sigmoid(-w) + 8) * 2.0**-24 + 2.0**-119


def _values(n):
    g = torch.Generator().manual_seed(n)
    v = torch.cat([torch.linspace(-13, 13, n // 2), torch.randn(n - n // 2, generator=g) * 0.3])
    return v[torch.randperm(n, generator=g)]


@pytest.mark.parametrize("rows,n", SIZES)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("res", [False, True])
def test_within_roundings(rows, n, act, gated, res):
    v = _values(n)
    bias = torch.cat([v, torch.ones(n)]) if gated else v
    x, w = torch.zeros(rows, 16, dtype=I8, device="cuda"), torch.ones(bias.numel(), 16, dtype=I8, device="cuda")
    got = linear_int8(x, w, torch.ones(bias.numel(), device="cuda"), bias.cuda(),
                      torch.zeros(rows, n, device="cuda") if res else None, x_scale=torch.ones(rows, device="cuda"),
                      activation=act, gated=gated, out_dtype=FP)
    assert bool((got == got[0]).all())
    want, tol = _want(v, act)
    off = (got[0].double().cpu() - want).abs() / tol
    assert float(off.max()) <= 1.0, f"{int((off > 1).sum())} off, worst {float(off.max()):.3f} at {float(v[off.argmax()])}"


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_far_values(act):
    inf = float("inf")
    v = torch.tensor([0.0, -0.0, 20.0, 1e10, 3e38, inf, -20.0, -1e10, -3e38, float("nan"), 1e-40, -1e-40])
    x, w = torch.zeros(40, 16, dtype=I8, device="cuda"), torch.ones(v.numel(), 16, dtype=I8, device="cuda")
    got = linear_int8(x, w, torch.ones(v.numel(), device="cuda"), v.cuda(), x_scale=torch.ones(40, device="cuda"),
                      activation=act, out_dtype=FP)[17].cpu()
    assert torch.equal(got[:6], torch.tensor([0.0, 0.0, 20.0, 1e10, 3e38, inf]))
    assert float(got[6:9].abs().max()) <= 5e-8 and not got[6:9].isnan().any() and bool(got[9].isnan())
    assert float((got[10:] - v[10:] / 2).abs().max()) <= 2.0**-148
