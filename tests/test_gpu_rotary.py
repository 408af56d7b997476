"""Rotary positions against the formula in 64 bits.

Bound of every element: the turn's own arithmetic is fp32, cosine and sine off by at
most 2^-21 (the reduced angle's rounding, then the function's) and three roundings of
2^-24 on top, so 2^-20 (|a| + |b|) amplitude covers it; the result is rounded once, half
a step of its type (or half of its smallest subnormal)."""

import math

import pytest
import torch

from late_interaction_kernels.encoder import attention_varlen, rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
SMALLEST = {BF: 2.0**-133, HF: 2.0**-24, FP: 2.0**-149}


def _turn64(x, pos, f, inter, amp, sign=1.0):
    """``x [..., heads, d]`` at ``pos [...]``, and the sum of the magnitudes that meet in each element."""
    x, r = x.double().cpu(), 2 * f.numel()
    t = (pos.double().cpu()[..., None] * f.double().cpu())[..., None, :]
    c, s = amp * torch.cos(t), amp * sign * torch.sin(t)
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if inter else (x[..., :r // 2], x[..., r // 2:r])
    ya, yb, m = a * c - b * s, b * c + a * s, a.abs() + b.abs()
    y, mass = x.clone(), torch.zeros_like(x)
    at = (slice(0, r, 2), slice(1, r, 2)) if inter else (slice(0, r // 2), slice(r // 2, r))
    for part, turned in zip(at, (ya, yb)):
        y[..., part], mass[..., part] = turned, m
    return y, mass * abs(amp)


def _check(got, want_mass):
    want, mass = want_mass
    g = got.detach().double().cpu()
    assert g.shape == want.shape
    tol = want.abs() * torch.finfo(got.dtype).eps / 2 + SMALLEST[got.dtype] / 2 + mass * 2.0**-20
    bad = (g - want).abs() > tol * (1 + 2.0**-10)  # (half a step of the rounded value, not of the exact one)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((g - want).abs() / tol).max())}"


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("n,length,h,hk,d,r", [
    (1, 1, 1, 1, 2, 2), (2, 33, 3, 1, 64, 64), (3, 7, 4, 2, 72, 72), (1, 130, 2, 2, 96, 24), (2, 5, 2, 1, 80, 50),
    (1, 300, 5, 5, 33, 6), (2, 9, 1, 3, 17, 16), (1, 3, 2, 1, 1024, 1024), (40, 41, 12, 12, 64, 64)])
def test_counted_positions(dtype, inter, n, length, h, hk, d, r):
    qkv = torch.randn(n, length, h + 2 * hk, d, device="cuda").to(dtype)
    q, k, _ = qkv.split([h, hk, hk], dim=2)
    f, _ = rotary_frequencies(r, device="cuda")
    yq, yk = rotary(q, k, frequencies=f, interleaved=inter, amplitude=1.25)
    pos = torch.arange(length).expand(n, -1)
    _check(yq, _turn64(q, pos, f, inter, 1.25))
    _check(yk, _turn64(k, pos, f, inter, 1.25))
    assert yq.is_contiguous() and yk.is_contiguous() and yq.dtype == dtype
    assert torch.equal(rotary(k, frequencies=f, interleaved=inter, amplitude=1.25), yk)


@pytest.mark.parametrize("pdtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("fdtype", [torch.float32, torch.float64])
def test_given_positions(pdtype, fdtype):
    n, length, h, d = 5, 19, 3, 64
    q = torch.randn(n, length, h, d, device="cuda")
    f = rotary_frequencies(d, 1e6, scaling="yarn", factor=8.0, original_length=4096, device="cuda")[0].to(fdtype)
    far = torch.randint(-2**31, 2**31 - 1, (n, 2 * length), device="cuda").to(pdtype)
    for pos in (far[:, ::2], far[:, :1].expand(n, length), far[0, :length], far[2, ::2]):
        _check(rotary(q, frequencies=f, positions=pos), _turn64(q, pos.expand(n, length), f, False, 1.0))
    flat = far.flatten()[:n * length]
    _check(rotary(q.flatten(0, 1), frequencies=f, positions=flat), _turn64(q.flatten(0, 1), flat, f, False, 1.0))


def test_far_positions_keep_their_phase():
    """At position p of frequency 1 an fp32 angle would be off by up to p 2^-24."""
    f = torch.tensor([1.0, 0.37], dtype=torch.float64, device="cuda")
    q = torch.tensor([1.0, 1.0, 0.0, 0.0], device="cuda").expand(1, 4, 1, 4)
    pos = torch.tensor([[0, 1 << 20, (1 << 31) - 1, -(1 << 31)]], device="cuda")
    got = rotary(q, frequencies=f, positions=pos).double().cpu()[0, :, 0]
    for i, p in enumerate(pos[0].tolist()):
        for j, w in enumerate(f.tolist()):
            tol = 2.0**-20 + abs(p) * w * 2.0**-50
            assert abs(float(got[i, j]) - math.cos(p * w)) <= tol and abs(float(got[i, j + 2]) - math.sin(p * w)) <= tol


@pytest.mark.parametrize("lens", [[1], [0, 3, 0, 0, 5, 1, 0], [64, 1, 130, 2], [1] * 300, []])
@pytest.mark.parametrize("before,behind", [(0, 0), (3, 4)])
def test_packed(lens, before, behind):
    tokens = before + sum(lens) + behind
    if tokens == 0:
        return
    q, k = torch.randn(tokens, 3, 40, device="cuda").to(BF), torch.randn(tokens, 1, 40, device="cuda").to(BF)
    outside = torch.ones(tokens, dtype=torch.bool)
    outside[before:before + sum(lens)] = False
    q[outside.cuda()] = float("nan")
    cu = torch.tensor([before] + lens, device="cuda").cumsum(0).int()
    f, _ = rotary_frequencies(40, device="cuda")
    pos = torch.cat([torch.zeros(before)] + [torch.arange(m) + 7 for m in lens] + [torch.zeros(behind)])
    q.requires_grad_()
    yq, yk = rotary(q, k, frequencies=f, cu_seqlens=cu, offset=7)
    (gq,) = torch.autograd.grad(yq, q, torch.full_like(yq, float("inf")).masked_fill(~outside.cuda()[:, None, None], 2.0))
    for y in (yq, yk, gq):
        assert torch.equal(y[outside.cuda()], torch.zeros_like(y[outside.cuda()]))
    on = ~outside
    _check(yq[on.cuda()], _turn64(q.detach()[on.cuda()], pos[on], f, False, 1.0))
    _check(yk[on.cuda()], _turn64(k[on.cuda()], pos[on], f, False, 1.0))
    two = torch.full_like(q.detach(), 2.0)[on.cuda()]
    _check(gq[on.cuda()], _turn64(two, pos[on], f, False, 1.0, -1.0))


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("inter", [False, True])
def test_gradients(dtype, inter):
    n, length, d, r = 2, 21, 48, 32
    f, amp = rotary_frequencies(r, scaling="yarn", factor=4.0, original_length=64, device="cuda")
    q = torch.randn(n, length, 4, d, device="cuda").to(dtype).requires_grad_()
    k = torch.randn(n, length, 2, d, device="cuda").to(dtype).requires_grad_()
    gq = torch.randn(n, 4, length, d, device="cuda").to(dtype).transpose(1, 2)
    gk = torch.randn(1, 1, 2, d, device="cuda").to(dtype).expand(n, length, 2, d)
    pos = torch.arange(length).expand(n, -1) - 4
    yq, yk = rotary(q, k, frequencies=f, offset=-4, interleaved=inter, amplitude=amp)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk), retain_graph=True)
    _check(dq, _turn64(gq, pos, f, inter, amp, -1.0))
    _check(dk, _turn64(gk, pos, f, inter, amp, -1.0))
    # one of the outputs only
    (only,) = torch.autograd.grad(yk, (k,), gk, retain_graph=True)
    assert torch.equal(only, dk)
    assert torch.autograd.grad(yk, (q,), gk, allow_unused=True, retain_graph=True)[0] is None
    # broadcast leaf: the sum of its copies' gradients
    base = torch.randn(1, length, 1, d, device="cuda").to(FP).requires_grad_()
    (db,) = torch.autograd.grad(rotary(base.expand(n, length, 4, d), frequencies=f, interleaved=inter), base,
                                gq.to(FP))
    want = _turn64(gq.float(), pos + 4, f, inter, 1.0, -1.0)[0].sum((0, 2), keepdim=True)
    assert float((db.double().cpu() - want).abs().max()) <= 8 * 8 * 2.0**-19  # 8 values of up to 8


def test_gradients_by_differences():
    f, _ = rotary_frequencies(16, device="cuda")
    q = torch.randn(1, 6, 2, 20, device="cuda", requires_grad=True)
    w = torch.randn(1, 6, 2, 20, device="cuda")

    def loss(x):
        return (rotary(x, frequencies=f, offset=100) * w).double().sum()

    (g,) = torch.autograd.grad(loss(q), q)
    u = torch.randn_like(q)
    with torch.no_grad():  # the map is linear: a step of 1 is exact but for roundings
        diff = float(loss(q + u) - loss(q - u)) / 2
    assert abs(diff - float((g.double() * u).sum())) <= 240 * 2.0**-16
    # and so is its derivative with respect to the gradient
    w.requires_grad_()
    (g,) = torch.autograd.grad((rotary(q, frequencies=f) * w).sum(), q, create_graph=True)
    (h,) = torch.autograd.grad((g * u).sum(), w)
    with torch.no_grad():
        assert float((h - rotary(u, frequencies=f)).abs().max()) <= 16 * 2.0**-20


def test_strides_and_empty():
    f, _ = rotary_frequencies(24, device="cuda")
    x = torch.randn(3, 2, 50, 11, device="cuda").to(HF)
    views = [x.permute(0, 3, 1, 2)[..., 1:25], x.permute(3, 0, 1, 2)[:2, :, :, ::2][..., :24],
             x[:, :, :24].permute(0, 3, 1, 2), torch.randn(1, 1, 1, 31, device="cuda").to(HF)[..., 3:30].expand(4, 5, 2, 27)]
    for v in views:
        pos = torch.arange(v.shape[1]).expand(v.shape[0], -1)
        _check(rotary(v, frequencies=f), _turn64(v, pos, f, False, 1.0))
    for shape in ((0, 4, 2, 24), (2, 0, 2, 24), (2, 4, 0, 24)):
        q = torch.randn(*shape, device="cuda", requires_grad=True)
        y = rotary(q, frequencies=f)
        assert y.shape == shape and torch.autograd.grad(y.sum(), q)[0].shape == shape
    q, k = torch.randn(2, 4, 0, 24, device="cuda"), torch.randn(2, 4, 3, 24, device="cuda")
    assert torch.equal(rotary(q, k, frequencies=f)[1], rotary(k, frequencies=f))


def test_other_stream_and_graph():
    f, _ = rotary_frequencies(64, device="cuda")
    q, k = (torch.randn(70, h, 64, device="cuda").to(BF) for h in (4, 2))
    cu = torch.tensor([0, 30, 70], dtype=torch.int32, device="cuda")
    want = rotary(q, k, frequencies=f, cu_seqlens=cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rotary(q, k, frequencies=f, cu_seqlens=cu)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rotary(q, k, frequencies=f, cu_seqlens=cu)
    for i in range(3):
        q.normal_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, rotary(q, k, frequencies=f, cu_seqlens=cu)))


def test_scores_depend_on_distances_only():
    """Attention over turned heads is the same wherever the sequences start."""
    f, _ = rotary_frequencies(64, device="cuda")
    q, k, v = (torch.randn(60, h, 64, device="cuda").to(HF) for h in (4, 2, 2))
    cu = torch.tensor([0, 25, 60], dtype=torch.int32, device="cuda")
    outs = []
    for offset in (0, 100000):
        a, b = rotary(q, k, frequencies=f, cu_seqlens=cu, offset=offset)
        outs.append(attention_varlen(a, b, v, cu, cu, 35, 35).double())
    # turned elements are off by 2^-11 of themselves: scores (64 terms of about 1, over 8) by about 2^-11,
    # probabilities by that share, outputs (|v| to 4) by 2^-8 at the most
    assert float((outs[0] - outs[1]).abs().max()) <= 2.0**-6
