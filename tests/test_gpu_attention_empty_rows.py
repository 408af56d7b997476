"""Queries that keep no key (a causal order over keys whose first ones are masked, a window past the last key) come out as
zeros and give no gradient, whatever they or their gradients hold."""

import pytest
import torch

from late_interaction_kernels.encoder import attention, attention_varlen

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
@pytest.mark.parametrize("size", [s for s in SIZES if s[0] == s[1]] + [(700, 700, 4, 1, 128)], ids=str)
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_queries_without_a_key(dtype, size, bad):
    """Causal with the first keys masked (padding in front): those queries come out as zeros, and a gradient that is not
    finite there (a normalised zero vector's, for one) reaches no other row."""
    print("[case]", dtype, size, bad, flush=True)
    L = size[0]
    q, k, v, gy = _make(3, *size, dtype)
    first = torch.tensor([9, L // 2, 0])
    km = torch.arange(L)[None] >= first[:, None]
    gy[~km] = 0
    clean = _grads(q, k, v, gy, None, km, causal=True)
    q[~km], gy[~km] = bad, bad
    for a, b in zip(_grads(q, k, v, gy, None, km, causal=True), clean):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("lq,lk,d", [(70, 30, 64), (150, 130, 64), (400, 350, 128)])
def test_queries_past_the_window(dtype, bad, packed, lq, lk, d):
    print("[case]", dtype, bad, packed, lq, lk, d, flush=True)
    q, k, v, gy = _make(1, lq, lk, 2, 2, d, dtype)
    none = slice(lk + 8, lq)
    gy[:, none] = 0

    def run():
        if not packed:
            return _grads(q, k, v, gy, None, None, window=8)
        ts = [t[0].cuda().requires_grad_() for t in (q, k, v)]
        cu = [torch.tensor([0, x], dtype=torch.int32).cuda() for x in (lq, lk)]
        out = attention_varlen(*ts, *cu, lq, lk, window=8)
        return [t.cpu() for t in (out.detach(), *torch.autograd.grad(out, ts, gy[0].cuda()))]

    clean = run()
    q[:, none], gy[:, none] = bad, bad
    for a, b in zip(run(), clean):
        assert torch.equal(a, b)
