"""Few queries over long keys: where the keys are split, and what that takes of memory."""

import ctypes

import pytest
import torch

from encoder_plain import ROUNDOFF, attention64, off
from late_interaction_kernels import _lib


def _size(n, lq, lk, h, hk, d):
    a = _lib.LikAttention(q=4096, k=4096, v=4096, dtype=_lib.LIK_BF16, heads=h, kv_heads=hk, dim=d, n=n, q_len=lq, k_len=lk,
                          q_stride_n=lq * h * d, q_stride_l=h * d, q_stride_h=d, k_stride_n=lk * hk * d, k_stride_l=hk * d,
                          k_stride_h=d, v_stride_n=lk * hk * d, v_stride_l=hk * d, v_stride_h=d, left=-1, right=-1, scale=0.1)
    return _lib.load().lik_attention_workspace_size(ctypes.byref(a))


@pytest.mark.parametrize("n", [1, 7, 60, 300, 4096, 20000])
@pytest.mark.parametrize("lq", [1, 5, 16, 64])
@pytest.mark.parametrize("lk", [256, 300, 1000, 9000])
@pytest.mark.parametrize("h,hk,d", [(12, 12, 64), (16, 4, 128), (8, 1, 64), (300, 300, 128)])
def test_workspace_stays_small(n, lq, lk, h, hk, d):
    """Partial sums of large batches are at most about a third of the keys' and values' bytes (with their statistics); of
    small ones some MB."""
    assert _size(n, lq, lk, h, hk, d) <= max(80 << 20, 0.36 * n * lk * hk * d * 4)


@pytest.mark.gpu
@pytest.mark.parametrize("n,lq,lk,h,hk,d", [
    (48, 64, 300, 12, 12, 64), (300, 1, 600, 4, 4, 64), (128, 1, 512, 4, 4, 64), (129, 1, 512, 4, 4, 64), (3, 10, 511, 2, 2, 64),
    (3, 11, 528, 2, 2, 64), (3, 11, 527, 2, 2, 64), (40, 5, 260, 8, 2, 64), (5, 16, 768, 16, 4, 128), (5, 16, 767, 16, 4, 128),
    (200, 2, 300, 8, 2, 128), (70, 1, 5000, 4, 4, 128)])
@pytest.mark.parametrize("masked", [False, True])
def test_both_sides_of_the_rule(n, lq, lk, h, hk, d, masked):
    from late_interaction_kernels.encoder import attention

    print("[case]", n, lq, lk, h, hk, d, masked, flush=True)
    g = torch.Generator().manual_seed(7)
    q = (torch.randn(n, lq, h, d, generator=g) * 1.5).to(torch.bfloat16)
    k, v = (torch.randn(n, lk, hk, d, generator=g).to(torch.bfloat16) for _ in range(2))
    km = torch.rand(n, lk, generator=g) < 0.7 if masked else torch.ones(n, lk, dtype=torch.bool)
    if masked:
        km[0], km[1, lk // 3:] = False, False
    got = attention(q.cuda(), k.cuda(), v.cuda(), None, km.cuda() if masked else None).cpu()
    some = [0, 1, 2, n // 2, n - 1]
    want = torch.stack([attention64(*(t[i].double() for t in (q, k, v)), km[i][None].expand(lq, -1), d**-0.5) for i in some])
    assert off(got[some], want) <= 1.25 * ROUNDOFF[torch.bfloat16]  # two roundings
    assert torch.isfinite(got).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_longest_mask_with_shared_heads(d):
    """As many keys as a mask may have, read by so many key heads that one workgroup takes large shares of them: their keep
    bits have to fit beside the tiles."""
    from late_interaction_kernels.encoder import attention

    lk, hk = 1 << 18, 300
    print("[case]", d, flush=True)
    g = torch.Generator().manual_seed(11)
    k, v = (torch.randn(1, lk, 1, d, generator=g).to(torch.bfloat16) for _ in range(2))
    km = torch.zeros(1, lk, dtype=torch.bool)
    km[0, :70] = km[0, lk // 2 - 9:lk // 2 + 50:2] = km[0, -40:] = True
    at = km[0].nonzero()[:, 0]
    q = (torch.randn(1, 1, 2 * hk, d, generator=g) * 1.5).to(torch.bfloat16)
    got = attention(q.cuda(), *(t.cuda().expand(-1, -1, hk, -1) for t in (k, v)), None, km.cuda()).cpu()
    want = attention64(q[0].double(), k[0, at].double(), v[0, at].double(), torch.ones(1, len(at)).bool(), d**-0.5)
    assert off(got[0], want) <= 1.25 * ROUNDOFF[torch.bfloat16]
