"""Packed rows that belong to no sequence: their outputs and gradients are zeros, not what
the memory held before, and the rows in sequences keep their bits."""

import pytest
import torch

from late_interaction_kernels.encoder import attention_varlen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("ql,kl,h,hk,d", [([70, 1, 200], [70, 1, 200], 2, 2, 64), ([300, 20], [300, 20], 4, 2, 64),
                                          ([1, 1, 1], [600, 700, 5], 4, 1, 128), ([200, 300], [400, 90], 2, 1, 128),
                                          ([0, 5], [3, 0], 2, 2, 40), ([700], [700], 2, 2, 64)])
@pytest.mark.parametrize("before,after", [(0, 300), (37, 0), (1, 1500)])
def test_rows_in_no_sequence_are_zeros(dtype, ql, kl, h, hk, d, before, after):
    print("[case]", dtype, ql, kl, h, hk, d, before, after, flush=True)
    g = torch.Generator().manual_seed(1)
    rows, keys = sum(ql), sum(kl)

    def make(n, heads):
        return torch.randn(n, heads, d, generator=g).to(dtype).cuda()

    q, gy = make(before + rows + after, h), make(before + rows + after, h)
    k, v = make(before + keys + after, hk), make(before + keys + after, hk)
    cu_q, cu_k = (torch.tensor([0] + x).cumsum(0).to(torch.int32).cuda() for x in (ql, kl))
    at_q, at_k = slice(before, before + rows), slice(before, before + keys)

    def run(q, k, v, gy, cu_q, cu_k):
        junk = [torch.full_like(t, float("nan")) for t in (q, q, k, v)]  # what the freed memory holds
        del junk
        ts = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        junk = [torch.full_like(t, float("nan")) for t in (q, q, k, v)]
        del junk
        out = attention_varlen(*ts, cu_q, cu_k, max(ql), max(kl))
        junk = [torch.full_like(t, float("nan")) for t in (q, k, v)]
        del junk
        return out.detach(), *torch.autograd.grad(out, ts, gy)

    got = run(q, k, v, gy, cu_q + before, cu_k + before)
    want = run(q[at_q], k[at_k], v[at_k], gy[at_q], cu_q, cu_k)
    for a, b, at in zip(got, want, (at_q, at_q, at_k, at_k)):
        assert torch.equal(a[at], b)
        a[at] = 0
        assert torch.equal(a, torch.zeros_like(a))


def test_no_sequence_at_all():
    q = torch.randn(9, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    for cu, most in (([0], 4), ([4], 4), ([3, 3, 3], 0)):
        c = torch.tensor(cu, dtype=torch.int32, device="cuda")
        out = attention_varlen(q, q, q, c, c, most, most)
        (g,) = torch.autograd.grad(out, q, torch.ones_like(out))
        assert torch.equal(out, torch.zeros_like(out)) and torch.equal(g, torch.zeros_like(g))
