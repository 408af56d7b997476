"""Queries that the mask drops come out as zeros whatever the kept values hold, also where a call's
keys are split and joined."""

import pytest
import torch

from late_interaction_kernels.encoder import attention

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("lq,lk,h,hk,d", [(4, 1000, 2, 2, 64), (1, 5000, 4, 1, 128), (40, 2000, 2, 2, 64), (200, 4000, 1, 1, 64),
                                          (130, 130, 2, 2, 64)])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan"), "lowest"])
@pytest.mark.parametrize("train", [False, True])
def test_zeros_beside_values_that_are_not_finite(lq, lk, h, hk, d, bad, train):
    print("[case]", lq, lk, h, hk, d, bad, train, flush=True)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(3, lq, h, d, generator=g).to(BF)
    k, v = (torch.randn(3, lk, hk, d, generator=g).to(BF) for _ in range(2))
    qm = torch.rand(3, lq, generator=g) < 0.5
    qm[0], qm[2] = False, True
    v[:, lk // 3] = torch.finfo(BF).min if bad == "lowest" else bad
    v[:, -1] = v[:, lk // 3]  # two lowest values: their sum passes the type's range
    ts = [t.cuda().requires_grad_(train) for t in (q, k, v)]
    out = attention(*ts, qm.cuda()).cpu()
    assert torch.equal(out[~qm], torch.zeros_like(out[~qm]))
    if bad != "lowest":
        assert not torch.isfinite(out[qm]).any()
