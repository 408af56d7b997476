"""Rows that lie further apart than the kernels' tile offsets reach are copied, not refused: the first token of long
sequences into the gated block, and attention over tensors whose batch lies inside their tokens."""

import pytest
import torch

from late_interaction_kernels.encoder import attention, gated_ffn

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("rows", [3, 130])
def test_gated_ffn_of_first_tokens(rows):
    d, f, apart = 64, 96, 2**21 + 64  # elements from one row to the next
    g = torch.Generator().manual_seed(1)
    wi, wo = (torch.randn(2 * f, d, generator=g) * 0.1).to(BF).cuda(), (torch.randn(d, f, generator=g) * 0.1).to(BF).cuda()
    far = torch.empty(rows, apart, dtype=BF, device="cuda")
    x, r, gy = (far[:, i * 64 : i * 64 + d] for i in range(3))
    for t in (x, r, gy):
        t.copy_(torch.randn(rows, d, generator=g))
    near = [t.contiguous() for t in (x, r, gy)]
    assert torch.equal(gated_ffn(x, wi, wo, r), gated_ffn(near[0], wi, wo, near[1]))
    res = []
    for x, r, gy in ((x, r, gy), near):
        ts = [t.detach().requires_grad_() for t in (x, wi, wo, r)]
        y = gated_ffn(*ts)
        res.append((y, *torch.autograd.grad(y, ts, gy)))
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_gated_ffn_of_far_weights():
    d, f, apart = 64, 8, 2**21 + 64
    g = torch.Generator().manual_seed(1)
    far = torch.empty(64, apart, dtype=BF, device="cuda")
    wi, wo = far[: 2 * f, :d], far[:, 64 : 64 + f]
    wi.copy_(torch.randn(2 * f, d, generator=g) * 0.1)
    wo.copy_(torch.randn(d, f, generator=g) * 0.1)
    x = torch.randn(40, d, generator=g).to(BF).cuda()
    gy = torch.randn(40, d, generator=g).to(BF).cuda()
    res = []
    for ws in ((wi, wo), (wi.contiguous(), wo.contiguous())):
        ts = [t.detach().requires_grad_() for t in (x, *ws)]
        y = gated_ffn(*ts)
        res.append((y, *torch.autograd.grad(y, ts, gy)))
    assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.parametrize("which", ["q", "k", "v", "gy"])
def test_attention_of_tokens_far_apart(which):
    L, d, apart = 70, 32, 2**24 + 64
    g = torch.Generator().manual_seed(2)
    near = {t: torch.randn(1, L, 1, d, generator=g).to(BF).cuda() for t in ("q", "k", "v", "gy")}
    far = torch.empty(L, apart, dtype=BF, device="cuda")[:, :d]
    far.copy_(near[which][0, :, 0])
    res = []
    for ts in ({**near, which: far[None, :, None]}, near):
        leaves = [ts[t].detach().requires_grad_() for t in "qkv"]
        out = attention(*leaves)
        res.append((out, *torch.autograd.grad(out, leaves, ts["gy"]), attention(*(ts[t] for t in "qkv"))))
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_one_row_inside_odd_ones():
    """A dimension of one element may have any stride: nothing steps over it."""
    g = torch.Generator().manual_seed(3)
    d, f = 64, 96
    wi, wo = (torch.randn(2 * f, d, generator=g) * 0.1).to(BF).cuda(), (torch.randn(d, f, generator=g) * 0.1).to(BF).cuda()
    wide = torch.randn(5, 100, generator=g).to(BF).cuda()
    x, r = wide[2:3, 36:], wide[4:5, 16:80]
    ts = [t.detach().requires_grad_() for t in (x, wi, wo, r)]
    us = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in (x, wi, wo, r)]
    gy = wide[0:1, 20:84]
    res = [(y, *torch.autograd.grad(y, ls, gy)) for ls in (ts, us) for y in (gated_ffn(*ls),)]
    assert all(torch.equal(a, b) for a, b in zip(*res))
    assert torch.equal(gated_ffn(x, wi, wo, r), res[0][0])
    # one head, one sequence, one query, each with a stride that is no multiple of 8
    flat = torch.randn(9 * 104, generator=g).to(BF).cuda()
    q = flat.as_strided((1, 1, 1, d), (3, 5, 7, 1))
    k, v = (flat.as_strided((1, 9, 1, d), (13, 104, 9, 1), at) for at in (0, 24))
    ts = [t.detach().requires_grad_() for t in (q, k, v)]
    us = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in (q, k, v)]
    gy = torch.randn(1, 1, 1, d, generator=g).to(BF).cuda()
    res = [(y, *torch.autograd.grad(y, ls, gy)) for ls in (ts, us) for y in (attention(*ls),)]
    assert all(torch.equal(a, b) for a, b in zip(*res))
    assert torch.equal(attention(q, k, v), res[0][0])


def test_no_rows_inside_odd_ones():
    """Keys of no rows, in a tensor whose rows are no multiple of 16 bytes apart, are no keys."""
    from late_interaction_kernels.encoder import attention_varlen

    q = torch.randn(5, 2, 64, device="cuda", dtype=BF, requires_grad=True)
    k = torch.randn(0, 2, 67, device="cuda", dtype=BF)[..., 3:].requires_grad_()
    cu_q, cu_k = (torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (5, 0))
    out = attention_varlen(q, k, k, cu_q, cu_k, 5, 9)
    gq, gk = torch.autograd.grad(out, (q, k), torch.ones_like(out))
    assert torch.equal(out, torch.zeros_like(out)) and torch.equal(gq, torch.zeros_like(gq)) and gk.shape == k.shape
    y = attention(q[None].detach(), k[None].detach(), k[None].detach())
    assert torch.equal(y, torch.zeros_like(y))
    x = torch.randn(0, 67, device="cuda", dtype=BF)[:, 3:].requires_grad_()
    wi, wo = torch.ones(96, 64, device="cuda", dtype=BF), torch.ones(64, 48, device="cuda", dtype=BF)
    (gx,) = torch.autograd.grad(gated_ffn(x, wi, wo, x).sum(), x)
    assert gx.shape == x.shape
