"""Gradients of attention over 129 to 320 keys, where one kernel walks a sequence's queries for all three, and just outside;
against the formula's in 64 bits. Bounds as for the other sizes: q and k 1.5 u (2 u with masks: rows of few keys), v 1.25 u."""

import pytest
import torch

from encoder_plain import ROUNDOFF, attention64, keep_pairs, off
from late_interaction_kernels.encoder import attention, attention_varlen

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def _make(n, lq, lk, h, hk, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(n, lq, h, d, generator=g) * 1.5).to(dtype)
    k, v = (torch.randn(n, lk, hk, d, generator=g).to(dtype) for _ in range(2))
    return q, k, v, torch.randn(n, lq, h, d, generator=g).to(dtype)


def _want(q, k, v, gy, keep, scale):
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    out = torch.stack([attention64(*(t[i] for t in leaves), keep[i], scale) for i in range(q.shape[0])])
    return torch.autograd.grad(out, leaves, torch.where(keep.any(2)[..., None, None], gy.double(), 0.0))


def _grads(q, k, v, gy, *masks, **kw):
    ts = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = attention(*ts, *(None if m is None else m.cuda() for m in masks), **kw)
    first = torch.autograd.grad(out, ts, gy.cuda(), retain_graph=True)
    for a, b in zip(first, torch.autograd.grad(out, ts, gy.cuda())):
        assert torch.equal(a, b)
    return first


def _compare(got, want, dtype, m=1.5):
    for name, a, b, f in zip("qkv", got, want, (m, m, 1.25)):
        assert torch.isfinite(a).all() and off(a, b) <= f * ROUNDOFF[dtype], name


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
@pytest.mark.parametrize("lq,lk,h,hk,d", [(129, 129, 2, 2, 64), (1, 192, 2, 2, 64), (33, 193, 2, 1, 8), (320, 320, 2, 2, 64),
                                          (321, 321, 2, 2, 64), (1024, 150, 2, 2, 32), (1025, 150, 2, 2, 32), (250, 300, 8, 2, 40),
                                          (40, 160, 32, 1, 64), (64, 257, 6, 3, 56), (200, 319, 2, 2, 128)])
def test_no_mask(dtype, lq, lk, h, hk, d):
    print("[case]", dtype, lq, lk, h, hk, d, flush=True)
    q, k, v, gy = _make(2, lq, lk, h, hk, d, dtype)
    keep = torch.ones(2, lq, lk, dtype=torch.bool)
    _compare(_grads(q, k, v, gy), _want(q, k, v, gy, keep, d**-0.5), dtype)


@pytest.mark.parametrize("causal,window", [(True, None), (False, 0), (False, 5), (False, 100), (True, 33), (False, 400)])
@pytest.mark.parametrize("lq,lk", [(180, 180), (300, 300), (500, 140), (90, 310)])
def test_causal_and_window(lq, lk, causal, window):
    print("[case]", lq, lk, causal, window, flush=True)
    q, k, v, gy = _make(2, lq, lk, 4, 2, 64, BF)
    keep = keep_pairs(lq, lk, causal, window)[None].expand(2, -1, -1)
    got = _grads(q, k, v, gy, causal=causal, window=window)
    want = _want(q, k, v, gy, keep, 0.125)
    if window == 0:  # one key a query: p is 1, the gradients of q and k are 0
        assert got[0].abs().max() <= 1e-4 and got[1].abs().max() <= 1e-4
        assert off(got[2], want[2]) <= 1.25 * ROUNDOFF[BF]
        return
    _compare(got, want, BF, 2.0)
    assert not got[0].cpu()[~keep.any(2)].any() and not got[1].cpu()[~keep.any(1)].any()


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
@pytest.mark.parametrize("lq,lk,h,hk,d", [(300, 300, 4, 2, 64), (170, 190, 2, 2, 32), (30, 310, 4, 1, 48)])
@pytest.mark.parametrize("which", ["both", "keys", "queries"])
def test_masks_and_what_they_hide(dtype, lq, lk, h, hk, d, which):
    """Prefixes, holes, whole blocks of 32 dropped in the middle, one token, none; masked rows may hold anything."""
    print("[case]", dtype, lq, lk, h, hk, d, which, flush=True)
    n = 7
    q, k, v, gy = _make(n, lq, lk, h, hk, d, dtype)
    g = torch.Generator().manual_seed(2)
    masks = []
    for length in (lq, lk):
        m = torch.rand(n, length, generator=g) < 0.6
        m[0] = True
        m[1] = torch.arange(length) < length // 3 + 1
        m[2] = False
        m[3] = torch.arange(length) == length - 1
        m[4, 10:-3] = False
        m[5, :length // 2] = False
        masks.append(m)
    qm, km = masks
    keep = (qm if which != "keys" else torch.ones_like(qm))[:, :, None] & (km if which != "queries" else torch.ones_like(km))[:, None, :]
    use = (qm if which != "keys" else None, km if which != "queries" else None)
    got = _grads(q, k, v, gy, *use)
    _compare(got, _want(q, k, v, gy, keep, d**-0.5), dtype, 2.0)
    if use[0] is not None:
        assert not got[0].cpu()[~qm].any()
    if use[1] is not None:
        assert not got[1].cpu()[~km].any() and not got[2].cpu()[~km].any()
    for bad in (float("nan"), float("-inf"), torch.finfo(dtype).max):
        ts = [t.clone() for t in (q, k, v, gy)]
        for t, m in zip(ts, (use[0], use[1], use[1], use[0])):
            if m is not None:
                t[~m] = bad
        for a, b in zip(_grads(*ts, *use), got):
            assert torch.equal(a, b)


def test_packed_and_strided():
    """Lengths from none to the bound, more keys than queries or fewer; rows inside a wider tensor; a gradient with strides."""
    g = torch.Generator().manual_seed(6)
    lq = torch.tensor([300, 0, 1, 64, 129, 33, 250, 7, 32, 31])
    lk = torch.tensor([300, 5, 0, 64, 200, 310, 1, 320, 33, 128])
    cq, ck = (torch.cat([torch.zeros(1, dtype=torch.long), x.cumsum(0)]).to(torch.int32) for x in (lq, lk))
    wide = torch.randn(int(cq[-1]), 3, 4, 64, generator=g).to(BF)
    kv = torch.randn(int(ck[-1]), 2, 2, 64, generator=g).to(BF)
    gy = torch.randn(4, int(cq[-1]), 64, generator=g).to(BF).transpose(0, 1)
    wc, kc = wide.cuda().requires_grad_(), kv.cuda().requires_grad_()
    out = attention_varlen(wc[:, 1], kc[:, 0], kc[:, 1], cq.cuda(), ck.cuda(), 300, 320)
    gw, gkv = torch.autograd.grad(out, (wc, kc), gy.cuda())
    for i in range(10):
        a, b, c, d = int(cq[i]), int(cq[i + 1]), int(ck[i]), int(ck[i + 1])
        leaves = [t.double().requires_grad_() for t in (wide[a:b, 1], kv[c:d, 0], kv[c:d, 1])]
        got = (gw[a:b, 1], gkv[c:d, 0], gkv[c:d, 1])
        if a == b or c == d:
            assert not any(t.any() for t in got)
            continue
        want = torch.autograd.grad(attention64(*leaves, torch.ones(b - a, d - c).bool(), 0.125), leaves, gy[a:b].double())
        if d - c == 1:
            assert got[0].abs().max() <= 1e-4 and got[1].abs().max() <= 1e-4
            assert off(got[2], want[2]) <= 1.25 * ROUNDOFF[BF]
            continue
        _compare(got, want, BF, 2.0)
