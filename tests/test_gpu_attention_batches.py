"""attention of many sequences of some hundred tokens (several rounds of the CUs, sequences that end inside tiles),
against the formula in 64 bits; bounds as for the other sizes: two roundings, 1.25 u."""

import pytest
import torch

from encoder_plain import ROUNDOFF, attention64, keep_pairs, off
from late_interaction_kernels.encoder import attention, attention_varlen

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def _make(n, lq, lk, h, hk, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(n, lq, h, d, generator=g) * 1.5).to(dtype)
    return q, *(torch.randn(n, lk, hk, d, generator=g).to(dtype) for _ in range(2))


def _check(got, q, k, v, keep, scale, dtype):
    some = [0, 1, 2, 3, len(q) // 2, len(q) - 1]
    want = torch.stack([attention64(*(t[i].double() for t in (q, k, v)), keep[i], scale) for i in some])
    assert off(got[some], want) <= 1.25 * ROUNDOFF[dtype]
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("lq,lk,h,hk,d,dtype", [(129, 129, 4, 4, 64, BF), (304, 304, 4, 2, 64, FP), (305, 305, 4, 4, 64, BF),
                                                (300, 300, 4, 1, 40, BF), (257, 192, 4, 4, 32, FP), (1, 200, 4, 4, 64, BF),
                                                (512, 303, 4, 4, 64, BF), (600, 256, 4, 4, 64, FP), (33, 289, 8, 8, 16, BF)])
@pytest.mark.parametrize("causal,window", [(False, None), (True, None), (False, 40), (True, 100)])
def test_no_mask(lq, lk, h, hk, d, dtype, causal, window):
    print("[case]", lq, lk, h, hk, d, dtype, causal, window, flush=True)
    q, k, v = _make(130, lq, lk, h, hk, d, dtype)
    keep = keep_pairs(lq, lk, causal, window)[None].expand(130, -1, -1)
    got = attention(q.cuda(), k.cuda(), v.cuda(), causal=causal, window=window)
    _check(got.cpu(), q, k, v, keep, d**-0.5, dtype)


@pytest.mark.parametrize("causal,window", [(False, None), (True, None), (False, 25)])
@pytest.mark.parametrize("holes", [False, True])
def test_masks_and_what_they_hide(holes, causal, window):
    print("[case]", holes, causal, window, flush=True)
    n, L = 140, 300
    q, k, v = _make(n, L, L, 4, 2, 64, BF)
    g = torch.Generator().manual_seed(3)
    m = torch.arange(L)[None] < torch.randint(1, L + 1, (n, 1), generator=g)
    if holes:
        m &= torch.rand(n, L, generator=g) < 0.7
    m[1], m[2] = False, True
    m[3] = torch.arange(L) == L - 1
    keep = m[:, :, None] & m[:, None, :] & keep_pairs(L, L, causal, window)
    got = attention(q.cuda(), k.cuda(), v.cuda(), m.cuda(), m.cuda(), causal=causal, window=window)
    _check(got.cpu(), q, k, v, keep, 0.125, BF)
    assert not got.cpu()[~keep.any(2)].any()
    for bad in (float("nan"), float("-inf"), torch.finfo(BF).max):
        q2, k2, v2 = q.clone(), k.clone(), v.clone()
        for t in (q2, k2, v2):
            t[~m] = bad
        again = attention(q2.cuda(), k2.cuda(), v2.cuda(), m.cuda(), m.cuda(), causal=causal, window=window)
        assert torch.equal(again, got)


def test_packed_and_gradients():
    """Packed rows with lengths from 0 to the bound; and a training step through the same forward."""
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 301, (150,), generator=g)
    lens[0], lens[1], lens[2], lens[3] = 300, 0, 1, 64
    cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).to(torch.int32)
    total = int(cu[-1])
    q, k, v, gy = (torch.randn(total, 4, 64, generator=g).to(BF) for _ in range(4))
    ts = [t.cuda().requires_grad_() for t in (q, k, v)]
    c = cu.cuda()
    out = attention_varlen(*ts, c, c, 300, 300, causal=True)
    grads = torch.autograd.grad(out, ts, gy.cuda())
    for i in (0, 2, 3, 75, 149):
        a, b = int(cu[i]), int(cu[i + 1])
        leaves = [t[a:b].double().requires_grad_() for t in (q, k, v)]
        want = attention64(*leaves, keep_pairs(b - a, b - a, True, None), 0.125)
        assert off(out[a:b], want) <= 1.25 * ROUNDOFF[BF]
        if b - a > 8:
            for x, y in zip(grads, torch.autograd.grad(want, leaves, gy[a:b].double())):
                assert off(x[a:b], y) <= 1.5 * ROUNDOFF[BF]
