"""Rows that a mask drops give and get no gradient, whatever the kept rows hold."""

import pytest
import torch

from late_interaction_kernels.encoder import attention

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16
SIZES = [(60, 60, 2, 2, 64), (150, 150, 4, 2, 64), (300, 300, 2, 2, 32), (100, 200, 2, 2, 128), (330, 330, 2, 1, 64)]


def _make(n, lq, lk, h, hk, d, dtype):
    g = torch.Generator().manual_seed(5)
    q, gy = (torch.randn(n, lq, h, d, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(n, lk, hk, d, generator=g).to(dtype) for _ in range(2))
    return q, k, v, gy


def _grads(q, k, v, gy, qm, km, **kw):
    ts = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = attention(*ts, *(None if m is None else m.cuda() for m in (qm, km)), **kw)
    return [t.cpu() for t in (out.detach(), *torch.autograd.grad(out, ts, gy.cuda()))]


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("which", ["k", "v", "both"])
def test_masked_queries_get_none(dtype, size, bad, which):
    """Kept keys and values that are not finite: the masked queries' gradients are zeros all the same; where
    every query is masked, so are those of k and v."""
    print("[case]", dtype, size, bad, which, flush=True)
    lq, lk = size[:2]
    q, k, v, gy = _make(3, *size, dtype)
    qm = torch.arange(lq)[None] < torch.tensor([lq // 2, 0, lq - 7])[:, None]
    if which != "v":
        k[:, lk // 2] = bad
    if which != "k":
        v[:, lk // 2] = bad
    out, gq, gk, gv = _grads(q, k, v, gy, qm, None)
    for t in (out, gq):
        assert torch.equal(t[~qm], torch.zeros_like(t[~qm]))
    for t in (gk, gv):
        assert torch.equal(t[1], torch.zeros_like(t[1]))


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
@pytest.mark.parametrize("size", [s for s in SIZES if s[0] == s[1]], ids=str)
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_keys_of_masked_queries_only(dtype, size, bad):
    """Causal: the last keys are kept by masked queries alone, and their values are not finite."""
    print("[case]", dtype, size, bad, flush=True)
    L = size[0]
    q, k, v, gy = _make(2, *size, dtype)
    qm = (torch.arange(L) < L - 9)[None].expand(2, -1)
    clean = _grads(q, k, v, gy, qm, None, causal=True)
    v[:, L - 4] = bad
    got = _grads(q, k, v, gy, qm, None, causal=True)
    for t in got[2:]:
        assert torch.equal(t[:, L - 9:], torch.zeros_like(t[:, L - 9:]))
    for t, c in zip(got[:2], clean):  # queries of other tiles never meet that value
        assert torch.equal(t[:, : L // 2 // 64 * 64], c[:, : L // 2 // 64 * 64])
