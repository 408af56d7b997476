"""fp16 attention: what lies between its products may leave fp16's range (largest value 65504, spacing
2^-24 at the lower end) although neither the inputs nor the results do.

Bounds: the output 1.25 u, the gradients of q and k 1.5 u and of v 1.25 u of the result's 2-norm, as at other sizes, and half a
spacing of 2^-24 an element for the rounding of the result itself."""

import pytest
import torch

from encoder_plain import ROUNDOFF, attention64
from late_interaction_kernels.encoder import attention

pytestmark = pytest.mark.gpu
FP = torch.float16


def _check(name, got, want, m):
    assert torch.isfinite(got).all(), name
    err = float((got.double().cpu() - want).norm())
    assert err <= m * ROUNDOFF[FP] * float(want.norm()) + 2.0**-25 * want.numel() ** 0.5, name


@pytest.mark.parametrize("lq,lk", [(1, 2048), (1, 131072), (100, 2048), (300, 300)])
def test_many_keys_far_below_the_largest(lq, lk):
    """One key has nearly all of the probability and a value of 0; the others share the rest, 2^-26 of it each, and their
    values are all of the output."""
    print("[case]", lq, lk, flush=True)
    d = 64
    q = torch.zeros(1, lq, 1, d)
    q[..., 0] = 1.0
    k = torch.zeros(1, lk, 1, d)
    k[0, lk // 2, 0, 0] = 26 * 0.6931471805599453
    v = torch.full((1, lk, 1, d), 2000.0)
    v[0, lk // 2] = 0
    q, k, v = (t.to(FP) for t in (q, k, v))
    want = attention64(q[0].double(), k[0].double(), v[0].double(), torch.ones(lq, lk).bool(), 1.0)
    _check("out", attention(q.cuda(), k.cuda(), v.cuda(), scale=1.0)[0], want, 1.25)


def _grads(q, k, v, gy, scale):
    n, lq, lk = q.shape[0], q.shape[1], k.shape[1]
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    keep = torch.ones(lq, lk, dtype=torch.bool)
    out = torch.stack([attention64(*(t[i] for t in leaves), keep, scale) for i in range(n)])
    want = torch.autograd.grad(out, leaves, gy.double())
    ts = [t.cuda().requires_grad_() for t in (q, k, v)]
    return torch.autograd.grad(attention(*ts, scale=scale), ts, gy.cuda()), want


@pytest.mark.parametrize("lq,lk,h,hk,d", [(200, 200, 2, 2, 64), (90, 90, 2, 1, 64), (150, 310, 4, 2, 32), (400, 400, 2, 2, 128)])
@pytest.mark.parametrize("size", [1e-4, 1e-3, 1e-2, 1.0, 1e3, 1e4])
def test_values_of_any_size(lq, lk, h, hk, d, size):
    print("[case]", lq, lk, h, hk, d, size, flush=True)
    g = torch.Generator().manual_seed(2)
    q = (torch.randn(2, lq, h, d, generator=g) * 1.5).to(FP)
    k = torch.randn(2, lk, hk, d, generator=g).to(FP)
    v = (torch.randn(2, lk, hk, d, generator=g).clamp(-4, 4) * size).to(FP)
    gy = (torch.randn(2, lq, h, d, generator=g) * min(1.0, 10 / size)).to(FP)
    got, want = _grads(q, k, v, gy, d**-0.5)
    for name, a, b, m in zip("qkv", got, want, (1.5, 1.5, 1.25)):
        _check(name, a, b, m)


@pytest.mark.parametrize("lk", [300, 20000, 100000])
def test_gradients_over_many_even_keys(lk):
    """Probabilities of about 1 / lk each. Their share of a gradient is small, the sums over the queries are not."""
    print("[case]", lk, flush=True)
    lq, d = 200, 16
    g = torch.Generator().manual_seed(3)
    q = (torch.randn(1, lq, 1, d, generator=g) * 0.1).to(FP)
    k, v = (torch.randn(1, lk, 1, d, generator=g).to(FP) for _ in range(2))
    gy = (torch.randn(1, lq, 1, d, generator=g) * 100).to(FP)
    got, want = _grads(q, k, v, gy, d**-0.5)
    for name, a, b, m in zip("qkv", got, want, (1.5, 1.5, 1.25)):
        _check(name, a, b, m)
