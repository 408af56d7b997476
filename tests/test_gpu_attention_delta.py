"""The gradients of q and k where delta = sum g o cancels against g v: values with a large common part. The forward keeps what
the output's rounding took off, so delta is as good as from fp32, and the output's weights are the rounded probabilities over
their own sum, so the common part comes out whole.

Bounds: with x = g v - delta of order s and a common part c of the values, what is left of the output's rounding in delta is at most
2^-8 of u c |g| sqrt(d) / s of x: under 0.1 u here, beside two roundings (ds, the gradient), so 1.25 u. Without the kept
byte that term is c / s = 16 times u."""

import pytest
import torch

from encoder_plain import ROUNDOFF, attention64, off
from late_interaction_kernels.encoder import attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("lq,lk,h,hk,d", [(64, 64, 2, 2, 64), (200, 200, 2, 1, 64), (130, 310, 2, 2, 32), (100, 400, 2, 2, 128),
                                          (16, 2000, 2, 2, 64)])
def test_common_part_of_the_values(dtype, lq, lk, h, hk, d):
    print("[case]", dtype, lq, lk, h, hk, d, flush=True)
    g = torch.Generator().manual_seed(9)
    q = (torch.randn(1, lq, h, d, generator=g) * 1.5).to(dtype)
    k = torch.randn(1, lk, hk, d, generator=g).to(dtype)
    sign = torch.randint(0, 2, (d,), generator=g) * 2 - 1.0
    v = (sign * 16 + torch.randn(1, lk, hk, d, generator=g)).to(dtype)
    gy = torch.randn(1, lq, h, d, generator=g).to(dtype)
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    out = attention64(*(t[0] for t in leaves), torch.ones(lq, lk).bool(), d**-0.5)[None]
    want = torch.autograd.grad(out, leaves, gy.double())
    ts = [t.cuda().requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(attention(*ts), ts, gy.cuda())
    for name, a, b in zip("qkv", got, want):
        assert off(a, b) <= 1.25 * ROUNDOFF[dtype], name
