"""Scores of any finite size: one key takes everything, and is the output's value to the roundings' bound (1.25 u of
the 2-norm for two of them), where a reference of 1e9 in fp32 is spaced by 64."""

import pytest
import torch

from encoder_plain import ROUNDOFF, attention64, off
from late_interaction_kernels.encoder import attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("lq,lk,h,hk,d", [(64, 64, 2, 2, 64), (4, 2000, 2, 2, 64), (1, 3000, 4, 1, 128), (150, 400, 2, 2, 40)])
@pytest.mark.parametrize("size", [300.0, 1e3, 3e3, 1e4, 3e4])
@pytest.mark.parametrize("masked", [False, True])
def test_one_key_takes_everything(dtype, lq, lk, h, hk, d, size, masked):
    print("[case]", dtype, lq, lk, h, hk, d, size, masked, flush=True)
    g = torch.Generator().manual_seed(1)
    q = (torch.randn(2, lq, h, d, generator=g).clamp(-2, 2) * size).to(dtype)
    k = (torch.randn(2, lk, hk, d, generator=g).clamp(-2, 2) * size).to(dtype)
    v = torch.randn(2, lk, hk, d, generator=g).to(dtype)
    km = torch.rand(2, lk, generator=g) < 0.6 if masked else torch.ones(2, lk, dtype=torch.bool)
    if masked:
        km[1, 5:] = False
    got = attention(q.cuda(), k.cuda(), v.cuda(), None, km.cuda() if masked else None)
    want = torch.stack([attention64(q[i].double(), k[i].double(), v[i].double(), km[i][None].expand(lq, -1), d**-0.5)
                        for i in range(2)])
    # fp32 products of d terms leave scores off by up to d 2^-24 of their size: where the two largest lie closer than 2^-10
    # of it the weights are not determined (a row of one key or none is)
    kept = km[:, None, None]
    s = torch.einsum("nqhd,nkhd->nhqk", q.double(), k.double().repeat_interleave(h // hk, 2))
    top = s.masked_fill(~kept, -1e30).topk(2, -1).values
    far = top[..., 0] - top[..., 1] > 2.0**-10 * s.masked_fill(~kept, 0).abs().amax(-1)
    sure = (far | (km.sum(1) < 2)[:, None, None]).transpose(1, 2)
    assert sure.any()
    assert off(got.cpu()[sure], want[sure]) <= 1.25 * ROUNDOFF[dtype]
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("lq,lk,h,hk,d", [(64, 64, 2, 2, 64), (4, 2000, 2, 2, 64), (150, 400, 2, 1, 40), (90, 300, 4, 2, 32),
                                          (64, 200, 2, 2, 128)])
@pytest.mark.parametrize("size", [300.0, 1e3, 1e4, 3e4])
def test_its_gradients(dtype, lq, lk, h, hk, d, size):
    """p is 1 and 0: the gradient of v is g of the rows that take each key (rounded once: u), and those of q and k vanish but for the
    fp32 rounding of g v - delta, d 2^-23 of their largest terms."""
    print("[case]", dtype, lq, lk, h, hk, d, size, flush=True)
    g = torch.Generator().manual_seed(2)
    q = (torch.randn(1, lq, h, d, generator=g).clamp(-2, 2) * size).to(dtype)
    k = (torch.randn(1, lk, hk, d, generator=g).clamp(-2, 2) * size).to(dtype)
    v = torch.randn(1, lk, hk, d, generator=g).to(dtype)
    s = torch.einsum("nqhd,nkhd->nhqk", q.double(), k.double().repeat_interleave(h // hk, 2))
    top = s.topk(2, -1).values
    sure = (top[..., 0] - top[..., 1] > 2.0**-10 * s.abs().amax(-1)).transpose(1, 2)
    assert sure.any()
    gy = torch.randn(1, lq, h, d, generator=g).to(dtype) * sure[..., None]  # (rows that are not determined: no gradient)
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    out = attention64(*(t[0] for t in leaves), torch.ones(lq, lk).bool(), d**-0.5)[None]
    want = torch.autograd.grad(out, leaves, gy.double())
    ts = [t.cuda().requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(attention(*ts), ts, gy.cuda())
    assert off(got[2], want[2]) <= ROUNDOFF[dtype]
    most = d * 2.0**-23 * float(gy.abs().max() * v.abs().max()) * d**-0.5
    assert float(got[0].double().abs().max()) <= most * float(k.abs().max())
    assert float(got[1].double().abs().max()) <= most * float(q.abs().max()) * (lq * h // hk)
