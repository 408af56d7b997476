"""Gradients under masks as long as they may be: the keep bits of 2^18 tokens beside the tiles, on either side."""

import pytest
import torch

from encoder_plain import ROUNDOFF, attention64, off
from late_interaction_kernels.encoder import attention

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("side", ["keys", "queries"])
def test_gradients(side, d):
    print("[case]", side, d, flush=True)
    long, few = 1 << 18, 70
    lq, lk = (few, long) if side == "keys" else (long, few)
    g = torch.Generator().manual_seed(1)
    q, gy = (torch.randn(1, lq, 1, d, generator=g).to(BF) for _ in range(2))
    k, v = (torch.randn(1, lk, 1, d, generator=g).to(BF) for _ in range(2))
    m = torch.zeros(1, long, dtype=torch.bool)
    m[0, 3:90] = m[0, long // 2 - 9:long // 2 + 50:2] = m[0, -40:] = True
    ts = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = attention(*ts, m.cuda() if side == "queries" else None, m.cuda() if side == "keys" else None)
    grads = torch.autograd.grad(out, ts, gy.cuda())
    at = m[0].nonzero()[:, 0]
    rows, cols = (slice(None), at) if side == "keys" else (at, slice(None))
    leaves = [q[0, rows].double().requires_grad_(), *(t[0, cols].double().requires_grad_() for t in (k, v))]
    want = attention64(*leaves, torch.ones(len(leaves[0]), len(leaves[1])).bool(), d**-0.5)
    ref = torch.autograd.grad(want, leaves, gy[0, rows].double())
    assert off(out[0, rows], want) <= 1.25 * ROUNDOFF[BF]  # two roundings; q and k three at most
    for got, r, i, f in zip(grads, ref, (rows, cols, cols), (1.5, 1.5, 1.25)):
        assert off(got[0, i], r) <= f * ROUNDOFF[BF]
        assert int((got != 0).any(-1).sum()) <= len(r)  # the others are zeros


def test_a_key_of_masked_queries_far_apart():
    """Causal: the last key's value is not finite and only masked queries, 2^18 of them, see it."""
    L, d = 1 << 18, 64
    g = torch.Generator().manual_seed(2)
    q, gy = (torch.randn(1, L, 1, d, generator=g).to(BF).cuda() for _ in range(2))
    k, v = (torch.randn(1, 200, 1, d, generator=g).to(BF).cuda() for _ in range(2))
    qm = (torch.arange(L) < 150)[None].cuda()
    qm[0, -1] = False
    v[0, 190] = float("nan")
    ts = [t.requires_grad_() for t in (q, k, v)]
    out = attention(*ts, qm, None, causal=True)
    _, gk, gv = torch.autograd.grad(out, ts, gy)
    assert not gk[0, 150:].any() and not gv[0, 150:].any()
