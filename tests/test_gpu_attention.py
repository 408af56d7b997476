"""attention / attention_varlen and their gradients against the formula in 64 bits.

Bounds: the output passes two roundings to the 16-bit type (the probabilities, the
output): sqrt(2 / 3) u in the 2-norm when errors spread evenly, bounded by 1.25 u.
The gradients of q and k pass three (the output in delta, ds, the gradient), bounded
by 1.5 u; where few keys share a row, delta's share grows to that of ds: 2 u for
sequences of a handful of keys. A gradient that is zero in the formula (one key a
row) is bounded by fp32 rounding of dp - delta, and by u of delta's terms through the
rounded output: u |g| |o|."""

import pytest
import torch

from encoder_plain import ROUNDOFF, attention64, keep_pairs, off
from late_interaction_kernels.encoder import attention, attention_varlen

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def _case(*tag):
    print("[case]", *tag, flush=True)


def _make(n, lq, lk, h, hk, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(n, lq, h, d, generator=g) * 1.5).to(dtype)
    k, v = (torch.randn(n, lk, hk, d, generator=g).to(dtype) for _ in range(2))
    return q, k, v, torch.randn(n, lq, h, d, generator=g).to(dtype)


def _want(q, k, v, gy, keep, scale):
    """Outputs and gradients of a batch, sequence by sequence; keep [n, lq, lk]."""
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    outs = [attention64(*(t[i] for t in leaves), keep[i], scale) for i in range(q.shape[0])]
    out = torch.stack(outs)
    seen = keep.any(2)[..., None, None]
    grads = torch.autograd.grad(out, leaves, torch.where(seen, gy.double(), 0.0))
    return out.detach(), grads


def _compare(got, grads, out, want, dtype, short=False):
    u = ROUNDOFF[dtype]
    assert off(got, out) <= 1.25 * u
    for name, a, b, m in zip("qkv", grads, want, (2.0 if short else 1.5, 2.0 if short else 1.5, 1.25)):
        assert off(a, b) <= m * u, name


def _run(q, k, v, gy, qm=None, km=None, **kw):
    ts = [t.cuda().requires_grad_() for t in (q, k, v)]
    qm, km = (None if m is None else m.cuda() for m in (qm, km))
    out = attention(*ts, qm, km, **kw)
    with torch.no_grad():
        assert torch.equal(out, attention(*ts, qm, km, **kw))
    return out, torch.autograd.grad(out, ts, gy.cuda())


SHAPES = [  # n, lq, lk, h, hk, d
    (2, 5, 5, 2, 2, 8), (1, 32, 32, 3, 3, 64), (2, 33, 33, 2, 1, 40), (2, 64, 64, 4, 2, 64), (1, 65, 65, 2, 2, 72),
    (2, 127, 127, 2, 2, 32), (1, 129, 129, 2, 2, 96), (2, 300, 300, 2, 2, 64), (1, 257, 257, 4, 1, 128),
    (1, 40, 300, 4, 4, 64), (2, 300, 40, 2, 2, 104), (1, 700, 700, 2, 2, 64),
]


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_no_mask(dtype, shape):
    _case(dtype, shape)
    n, lq, lk, h, hk, d = shape
    q, k, v, gy = _make(*shape, dtype)
    keep = torch.ones(n, lq, lk, dtype=torch.bool)
    out, want = _want(q, k, v, gy, keep, d**-0.5)
    _compare(*_run(q, k, v, gy), out, want, dtype, lk <= 8)


@pytest.mark.parametrize("causal,window", [(True, None), (False, 0), (False, 3), (False, 70), (True, 16),
                                           (False, 1 << 20)])
@pytest.mark.parametrize("lq,lk", [(50, 50), (300, 300), (200, 90), (90, 200)])
def test_causal_and_window(causal, window, lq, lk):
    _case(causal, window, lq, lk)
    q, k, v, gy = _make(2, lq, lk, 4, 2, 64, BF)
    keep = keep_pairs(lq, lk, causal, window)[None].expand(2, -1, -1)
    out, want = _want(q, k, v, gy, keep, 0.2)
    got, grads = _run(q, k, v, gy, causal=causal, window=window, scale=0.2)
    if window == 0:  # one key a row: the output is its value, dv is g, and dq and dk vanish
        m = min(lq, lk)
        assert torch.equal(got[:, :m].cpu(), v[:, :m].repeat_interleave(2, 2))
        assert not got[:, m:].any() and off(grads[2], want[2]) <= 1.25 * ROUNDOFF[BF]
        assert grads[0].abs().max() <= 1e-4 and grads[1].abs().max() <= 1e-4
        return
    _compare(got, grads, out, want, BF, short=window == 3)


def _masks(n, lq, lk, seed):
    """Prefixes, holes, single tokens, one empty and one full row."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for length in (lq, lk):
        m = torch.rand(n, length, generator=g) < 0.6
        m[0] = True
        m[1] = torch.arange(length) < length // 3 + 1
        if n > 3:
            m[2] = False
            m[3] = torch.arange(length) == length - 1
        out.append(m)
    return out


@pytest.mark.parametrize("dtype,shape", [(BF, (6, 70, 70, 2, 2, 64)), (FP, (6, 300, 300, 4, 2, 64)),
                                         (BF, (5, 130, 200, 2, 1, 128)), (FP, (5, 33, 64, 2, 2, 72)),
                                         (BF, (4, 1, 500, 4, 2, 64)), (BF, (4, 9, 1, 2, 2, 32))], ids=str)
@pytest.mark.parametrize("which", ["both", "keys", "queries"])
def test_masks(dtype, shape, which):
    _case(dtype, shape, which)
    n, lq, lk, h, hk, d = shape
    q, k, v, gy = _make(*shape, dtype)
    qm, km = _masks(n, lq, lk, 3)
    qm, km = (None if which == "keys" else qm), (None if which == "queries" else km)
    keep = torch.ones(n, lq, lk, dtype=torch.bool)
    if qm is not None:
        keep = keep & qm[:, :, None]
    if km is not None:
        keep = keep & km[:, None, :]
    out, want = _want(q, k, v, gy, keep, d**-0.5)
    got, grads = _run(q, k, v, gy, qm, km)
    if lk == 1:
        assert off(got, out) <= 1.25 * ROUNDOFF[dtype] and off(grads[2], want[2]) <= 1.25 * ROUNDOFF[dtype]
        assert grads[0].abs().max() <= 1e-4 and grads[1].abs().max() <= 1e-4
        return
    _compare(got, grads, out, want, dtype, short=True)
    assert not got.cpu()[~keep.any(2)].any()
    if qm is not None:
        assert not grads[0].cpu()[~qm].any()
    if km is not None:
        assert not grads[1].cpu()[~km].any() and not grads[2].cpu()[~km].any()


@pytest.mark.parametrize("causal,window", [(False, None), (True, None), (False, 20)])
def test_nothing_of_masked_rows_is_used(causal, window):
    """NaN, infinities and the type's lowest value in masked rows of q, k, v and the gradient."""
    q, k, v, gy = _make(4, 150, 150, 2, 1, 64, BF)
    qm, km = _masks(4, 150, 150, 9)
    clean = _run(q, k, v, gy, qm, km, causal=causal, window=window)
    for bad in (float("nan"), float("inf"), torch.finfo(BF).min):
        q2, k2, v2, g2 = q.clone(), k.clone(), v.clone(), gy.clone()
        q2[~qm], g2[~qm], k2[~km], v2[~km] = bad, bad, bad, bad
        got = _run(q2, k2, v2, g2, qm, km, causal=causal, window=window)
        assert torch.equal(got[0], clean[0])
        assert all(torch.equal(a, b) for a, b in zip(got[1], clean[1]))


def test_other_masks_types_and_broadcast():
    q, k, v, gy = _make(3, 60, 80, 2, 2, 64, FP)
    km = torch.arange(80) < 50
    ref = _run(q, k, v, gy, None, km[None].expand(3, 80))
    for m in (km[None].expand(3, 80).to(torch.uint8), km[None].repeat(3, 1).long(), km[None].repeat(3, 1).float(),
              torch.stack([km, km, km], 1).t()):
        got = _run(q, k, v, gy, None, m)
        assert torch.equal(got[0], ref[0]) and all(torch.equal(a, b) for a, b in zip(got[1], ref[1]))


@pytest.mark.parametrize("dtype,h,hk,d", [(BF, 2, 2, 64), (FP, 4, 1, 128), (BF, 2, 1, 72)], ids=str)
@pytest.mark.parametrize("causal,window", [(False, None), (True, None), (False, 30)])
def test_packed(dtype, h, hk, d, causal, window):
    lens = [1, 64, 0, 200, 33, 129, 2]
    _case(dtype, h, hk, d, causal, window)
    g = torch.Generator().manual_seed(2)
    total = sum(lens)
    q = torch.randn(total, h, d, generator=g).to(dtype)
    k, v = (torch.randn(total, hk, d, generator=g).to(dtype) for _ in range(2))
    gy = torch.randn(total, h, d, generator=g).to(dtype)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    out = torch.cat([attention64(*(t[a:b] for t in leaves), keep_pairs(b - a, b - a, causal, window), d**-0.5)
                     for a, b in zip(cu.tolist(), cu.tolist()[1:]) if b > a])
    want = torch.autograd.grad(out, leaves, gy.double())
    ts = [t.cuda().requires_grad_() for t in (q, k, v)]
    c = cu.cuda()
    got = attention_varlen(*ts, c, c, 200, 300, causal=causal, window=window)
    with torch.no_grad():
        assert torch.equal(got, attention_varlen(*ts, c.long(), c, causal=causal, window=window))
    _compare(got, torch.autograd.grad(got, ts, gy.cuda()), out.detach(), want, dtype)


def test_packed_cross():
    """Different lengths on both sides, among them sequences without queries or without keys."""
    ql, kl, h, d = [3, 0, 40, 5], [70, 10, 0, 300], 2, 64
    g = torch.Generator().manual_seed(2)
    q, gy = (torch.randn(sum(ql), h, d, generator=g).to(BF) for _ in range(2))
    k, v = (torch.randn(sum(kl), h, d, generator=g).to(BF) for _ in range(2))
    cq, ck = (torch.tensor([0] + x).cumsum(0).to(torch.int32) for x in (ql, kl))
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    outs = []
    for i in range(4):
        a, b, x, y = cq[i], cq[i + 1], ck[i], ck[i + 1]
        if b > a:
            outs.append(attention64(leaves[0][a:b], leaves[1][x:y], leaves[2][x:y], torch.ones(b - a, y - x).bool(), 0.125)
                        if y > x else torch.zeros(b - a, h, d, dtype=torch.float64))
    out = torch.cat(outs)
    want = torch.autograd.grad(out, leaves, gy.double())
    ts = [t.cuda().requires_grad_() for t in (q, k, v)]
    got = attention_varlen(*ts, cq.cuda(), ck.cuda())
    grads = torch.autograd.grad(got, ts, gy.cuda())
    _compare(got, grads, out.detach(), want, BF)
    assert not got[3:43].any() and not grads[0][3:43].any() and not grads[1][70:80].any()


@pytest.mark.parametrize("n,lq,lk,h,hk,d", [(1, 1, 5000, 4, 1, 128), (3, 1, 2000, 2, 2, 64), (2, 7, 4097, 8, 2, 64),
                                            (1, 16, 1025, 2, 1, 72), (1, 40, 3000, 2, 2, 64)])
def test_few_rows_over_long_keys(n, lq, lk, h, hk, d):
    _case(n, lq, lk, h, hk, d)
    q, k, v, gy = _make(n, lq, lk, h, hk, d, BF)
    km = torch.rand(n, lk, generator=torch.Generator().manual_seed(4)) < 0.5
    km[0, lk // 5:] = False  # whole splits without a key
    keep = km[:, None, :].expand(n, lq, lk)
    out, want = _want(q, k, v, gy, keep, d**-0.5)
    _compare(*_run(q, k, v, gy, None, km), out, want, BF)
    none = attention(q.cuda(), k.cuda(), v.cuda(), None, torch.zeros_like(km).cuda())
    assert not none.any()


def test_peaked_and_large_scores():
    """Scores far apart: one key takes everything; and rows whose running maximum keeps growing."""
    q, k, v, gy = _make(1, 100, 400, 2, 2, 64, BF)
    k = (k.float() * torch.linspace(0.1, 12, 400)[None, :, None, None]).to(BF)
    keep = torch.ones(1, 100, 400, dtype=torch.bool)
    out, want = _want(q, k, v, gy, keep, 0.5)
    got, grads = _run(q, k, v, gy, scale=0.5)
    # fp32 scores of size up to s carry 2^-24 s of error, e^s then that share of p: well under u here
    _compare(got, grads, out, want, BF, short=True)


@pytest.mark.parametrize("size", [1e-4, 1.0, 100.0])
def test_fp16_gradients_of_any_size(size):
    """Small gradients are not lost in fp16's range on the way (they are as exact as its outputs allow)."""
    q, k, v, gy = _make(1, 200, 200, 2, 2, 64, FP)
    gy = (gy.float() * size).to(FP)
    keep = torch.ones(1, 200, 200, dtype=torch.bool)
    out, want = _want(q, k, v, gy, keep, 0.125)
    got, grads = _run(q, k, v, gy)
    for a, b in zip(grads, want):
        # besides the relative bound, fp16 outputs have a spacing of 2^-24
        b = b.to(FP).double()
        err = (a.double().cpu() - b).norm()
        assert err <= 1.5 * ROUNDOFF[FP] * b.norm() + 2.0**-24 * b.numel() ** 0.5


def test_gradient_against_differences():
    q, k, v, gy = _make(1, 40, 50, 2, 1, 32, FP)
    ts = [t.cuda().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(attention(*ts), ts, gy.cuda())
    g = torch.Generator().manual_seed(5)
    keep = torch.ones(40, 50, dtype=torch.bool)
    for i, grad in enumerate(grads):
        w = torch.randn(grad.shape, generator=g, dtype=torch.float64)

        def f(step):
            a = [t.double() for t in (q, k, v)]
            a[i] = a[i] + step * w
            return (attention64(*(t[0] for t in a), keep, 32**-0.5) * gy[0].double()).sum()

        want = float((f(1e-5) - f(-1e-5)) / 2e-5)
        bound = 4 * ROUNDOFF[FP] * float(grad.double().norm().cpu() * w.norm()) / w.numel() ** 0.5
        assert abs(float((grad.double().cpu() * w).sum()) - want) <= bound


def test_strides_odd_head_dims_and_order():
    n, L, h, d = 2, 140, 3, 64
    g = torch.Generator().manual_seed(7)
    qkv = torch.randn(n, L, 3, h, d, generator=g).to(BF).cuda()
    gy = torch.randn(n, L, h, d, generator=g).to(BF).cuda()
    parts = [qkv[:, :, i].detach().requires_grad_() for i in range(3)]
    whole = [t.detach().contiguous().requires_grad_() for t in parts]
    heads_first = [t.detach().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_() for t in parts]
    res = []
    for ts in (parts, whole, heads_first, whole):
        out = attention(*ts)
        res.append([out, *torch.autograd.grad(out, ts, gy)])
    g2 = gy.transpose(1, 2).contiguous().transpose(1, 2)
    out = attention(*whole)
    res.append([out, *torch.autograd.grad(out, whole, g2)])
    for other in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(res[0], other))
    q, k, v, gy = _make(2, 50, 50, 2, 2, 20, FP)  # a head dim that is padded
    keep = torch.ones(2, 50, 50, dtype=torch.bool)
    out, want = _want(q, k, v, gy, keep, 20**-0.5)
    _compare(*_run(q, k, v, gy), out, want, FP)


def test_only_some_gradients_and_broadcast_inputs():
    q, k, v, gy = (t.cuda() for t in _make(2, 70, 70, 2, 2, 64, BF))
    ts = [t.clone().requires_grad_() for t in (q, k, v)]
    full = torch.autograd.grad(attention(*ts), ts, gy)
    for i in range(3):
        one = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        (g,) = torch.autograd.grad(attention(*one), [one[i]], gy)
        assert torch.equal(g, full[i])
    # keys shared by the batch: the gradient of the broadcast input is the batch's sum
    kb, vb = (t[:1].clone().requires_grad_() for t in (k, v))
    out = attention(q, kb.expand(2, -1, -1, -1), vb.expand(2, -1, -1, -1))
    gk, gv = torch.autograd.grad(out, (kb, vb), gy)
    kk, vv = (t[:1].repeat(2, 1, 1, 1).requires_grad_() for t in (k, v))
    gk2, gv2 = torch.autograd.grad(attention(q, kk, vv), (kk, vv), gy)
    assert off(gk, gk2.double().sum(0, keepdim=True)) <= ROUNDOFF[BF]
    assert off(gv, gv2.double().sum(0, keepdim=True)) <= ROUNDOFF[BF]


def test_empty_calls():
    for n, lq, lk in ((0, 4, 4), (2, 0, 5), (2, 5, 0)):
        q = torch.randn(n, lq, 2, 16, device="cuda", dtype=BF, requires_grad=True)
        k, v = (torch.randn(n, lk, 2, 16, device="cuda", dtype=BF, requires_grad=True) for _ in range(2))
        out = attention(q, k, v)
        assert out.shape == q.shape and not out.any()
        for g, t in zip(torch.autograd.grad(out, (q, k, v), torch.ones_like(out)), (q, k, v)):
            assert g.shape == t.shape and not g.any()


def test_long_masked_keys():
    """One query over 100,000 keys of which the last ones are kept."""
    lk = 100_000
    q, k, v, _ = _make(1, 1, lk, 1, 1, 16, BF)
    km = torch.zeros(1, lk, dtype=torch.bool)
    km[0, -300:] = True
    want = attention64(q[0].double(), k[0, -300:].double(), v[0, -300:].double(), torch.ones(1, 300).bool(), 0.25)
    got = attention(q.cuda(), k.cuda(), v.cuda(), None, km.cuda())
    assert off(got[0], want) <= 1.25 * ROUNDOFF[BF]


@pytest.mark.parametrize("lk", [1 << 17, (1 << 17) + 33, 1 << 18])
@pytest.mark.parametrize("d", [64, 128])
def test_longest_masks_with_many_heads(lk, d):
    """As many keys as a mask may have, read by so many heads that a workgroup takes large shares of them: few rows
    and a tile of rows. The heads' keys are one tensor."""
    _case(lk, d)
    h = 300
    g = torch.Generator().manual_seed(11)
    k, v = (torch.randn(1, lk, 1, d, generator=g).to(BF) for _ in range(2))
    km = torch.zeros(1, lk, dtype=torch.bool)
    km[0, :70] = km[0, lk // 2 - 9:lk // 2 + 50:2] = km[0, -40:] = True
    at = km[0].nonzero()[:, 0]
    for lq in (1, 66):
        q = (torch.randn(1, lq, h, d, generator=g) * 1.5).to(BF)
        got = attention(q.cuda(), *(t.cuda().expand(-1, -1, h, -1) for t in (k, v)), None, km.cuda()).cpu()
        want = attention64(q[0].double(), k[0, at].double(), v[0, at].double(), torch.ones(lq, len(at)).bool(), d**-0.5)
        assert off(got[0], want) <= 1.25 * ROUNDOFF[BF]


def test_side_stream():
    q, k, v, gy = (t.cuda() for t in _make(2, 300, 300, 2, 2, 64, BF))
    want = attention(q, k, v)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = attention(q * 2 - q, k, v)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
