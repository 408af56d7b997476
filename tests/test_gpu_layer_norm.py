"""layer_norm and its gradients against the formula in 64 bits.

Bounds: y and grad_x are fp32 results rounded once, so off by at most the type's
roundoff; fp32 ones by their arithmetic: rows of at most 8192 terms are summed in
trees and chains of at most 32 + 8 additions, each relative 2^-24, and so are up to
700 rows of the weights' gradients: 64 * 2^-24 with room for the mean's
cancellation. 16-bit weights' gradients are rounded once more."""

import pytest
import torch

from encoder_plain import ROUNDOFF, layer_norm64, off
from late_interaction_kernels.encoder import layer_norm

pytestmark = pytest.mark.gpu
FP32 = 64 * 2.0**-24


def _case(*tag):
    print("[case]", *tag, flush=True)


def _make(rows, d, dtype, wdtype, bias, residual, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, d, generator=g) * 1.5 + 0.5).to(dtype)
    w = (torch.randn(d, generator=g) * 0.2 + 1).to(wdtype)
    b = (torch.randn(d, generator=g) * 0.2).to(wdtype) if bias else None
    r = torch.randn(rows, d, generator=g).to(dtype) if residual else None
    gy = torch.randn(rows, d, generator=g).to(dtype)
    gs = torch.randn(rows, d, generator=g).to(dtype) if residual else None
    return x, w, b, r, gy, gs


def _run64(x, w, b, r, gy, gs, eps, dtype):
    x, w, b, r, gy, gs = (None if t is None else t.double() for t in (x, w, b, r, gy, gs))
    total = x if r is None else (x + r).to(dtype).double()
    leaves = [t.requires_grad_() for t in (total, w, b) if t is not None]
    y, _ = layer_norm64(total, w, b, None, eps, None)
    grads = list(torch.autograd.grad(y, leaves, gy))
    if gs is not None:
        grads[0] = grads[0] + gs
    return y.detach(), total.detach(), grads


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 8), (3, 7), (5, 64), (2, 129), (33, 768), (7, 1027), (64, 1024),
                                    (9, 2050), (4, 4095), (3, 8192), (700, 40)])
@pytest.mark.parametrize("wide,bias,residual", [(True, True, True), (False, True, False), (True, False, False),
                                                (False, False, True)])
def test_values_and_gradients(dtype, rows, d, wide, bias, residual):
    _case(dtype, rows, d, wide, bias, residual)
    wdtype = torch.float32 if wide else dtype
    x, w, b, r, gy, gs = _make(rows, d, dtype, wdtype, bias, residual)
    y64, s64, g64 = _run64(x, w, b, r, gy, gs, 1e-5, dtype)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    xs, ws, bs, rs = (next(it) if t is not None else None for t in (x, w, b, r))
    out = layer_norm(xs, ws, bs, rs, eps=1e-5)
    with torch.no_grad():  # the inference path gives the same bits
        again = layer_norm(xs, ws, bs, rs, eps=1e-5)
    y, total = out if residual else (out, None)
    assert torch.equal(y, again[0] if residual else again)
    u = max(ROUNDOFF[dtype], FP32)
    # a single value has no deviation: its norm is the bias (or 0) up to cancellation
    if d > 1:
        assert off(y, y64) <= u
    else:
        assert (y.double().cpu() - y64).abs().max() <= u * max(1.0, float(y64.abs().max()))
    if residual:
        assert torch.equal(total.double().cpu(), s64)
        assert torch.equal(again[1], total)
    grads = torch.autograd.grad((y, total) if residual else (y,), leaves,
                                (gy.cuda(), gs.cuda()) if residual else (gy.cuda(),))
    got = dict(zip([n for n, t in zip("xwbr", (x, w, b, r)) if t is not None], grads))
    want = dict(zip([n for n, t in zip("xwb", (x, w, b)) if t is not None], g64))
    uw = max(ROUNDOFF[wdtype], FP32)
    if d > 1:
        assert off(got["x"], want["x"]) <= u
        assert off(got["w"], want["w"]) <= uw
    else:  # gradients of nothing: zeros, and the sum's own gradient
        assert (got["x"].double().cpu() - want["x"]).abs().max() <= u * 4
        assert (got["w"].double().cpu() - want["w"]).abs().max() <= uw * 4
    if bias:
        assert off(got["b"], want["b"]) <= uw
    if residual:
        assert torch.equal(got["x"], got["r"])


def test_gradient_against_differences():
    """The kernel's gradient along a direction against central differences of the formula."""
    x, w, b, r, gy, gs = _make(6, 50, torch.float32, torch.float32, True, False)
    xs, ws, bs = (t.cuda().requires_grad_() for t in (x, w, b))
    gx, gw, gb = torch.autograd.grad(layer_norm(xs, ws, bs), (xs, ws, bs), gy.cuda())
    g = torch.Generator().manual_seed(5)
    for t, grad in ((x, gx), (w, gw), (b, gb)):
        v = torch.randn(t.shape, generator=g, dtype=torch.float64)
        h = 1e-5

        def f(step):
            a = {id(x): x.double(), id(w): w.double(), id(b): b.double()}
            a[id(t)] = t.double() + step * v
            return (layer_norm64(a[id(x)], a[id(w)], a[id(b)], None, 1e-5, None)[0] * gy.double()).sum()

        want = float((f(h) - f(-h)) / (2 * h))  # truncation ~ h^2, rounding ~ 1e-16 / h: both under 1e-8
        size = float(grad.double().norm().cpu() * v.norm())
        assert abs(float((grad.double().cpu() * v).sum()) - want) <= 1e-5 * size


def test_many_rows_strides_and_order():
    """More rows than one round of the backward's workgroups, rows inside wider ones, other leading dims,
    and the same bits twice."""
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(9000, 130, generator=g).to(torch.bfloat16).cuda()
    x = wide[:, 3:99]  # rows start on odd elements
    w = (torch.randn(96, generator=g) * 0.1 + 1).cuda()
    gy = torch.randn(9000, 96, generator=g).to(torch.bfloat16).cuda()
    xs, ws = x.detach().requires_grad_(), w.requires_grad_()
    y = layer_norm(xs, ws)
    y64, _, (gx64, gw64) = _run64(x.cpu(), w.detach().cpu(), None, None, gy.cpu(), None, 1e-5, torch.bfloat16)
    assert off(y, y64) <= ROUNDOFF[torch.bfloat16]
    first = torch.autograd.grad(layer_norm(xs, ws), (xs, ws), gy)
    second = torch.autograd.grad(layer_norm(xs, ws), (xs, ws), gy)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    assert off(first[0], gx64) <= ROUNDOFF[torch.bfloat16]
    assert off(first[1], gw64) <= 1e-5  # 9000 rows: up to 1024 slices of 9 rows, summed in 16 chains of 64
    three = layer_norm(x.contiguous().view(90, 100, 96), ws)
    assert torch.equal(three.view(9000, 96), layer_norm(x.contiguous(), ws))


def test_non_finite_rows_stay_apart_and_empty_calls():
    x = torch.randn(5, 100, device="cuda")
    x[1, 3] = float("nan")
    x[2, 4] = float("inf")
    w = torch.ones(100, device="cuda")
    y = layer_norm(x, w)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).any()
    assert torch.isfinite(y[[0, 3, 4]]).all()
    e = torch.empty(0, 100, device="cuda", requires_grad=True)
    w.requires_grad_()
    y = layer_norm(e, w)
    gx, gw = torch.autograd.grad(y, (e, w), torch.empty(0, 100, device="cuda"))
    assert y.shape == (0, 100) and gx.shape == (0, 100) and torch.equal(gw, torch.zeros_like(w))


def test_only_the_sum_is_used():
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    r = torch.randn(4, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    _, s = layer_norm(x, w, None, r)
    gx, gw, gr = torch.autograd.grad(s.sum(), (x, w, r))
    assert torch.equal(gx, torch.ones_like(x)) and torch.equal(gr, gx) and torch.equal(gw, torch.zeros_like(w))


def test_side_stream():
    x = torch.randn(512, 768, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(768, device="cuda")
    want = layer_norm(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = (x * 2 - x)  # made on the stream that the call uses
        got = layer_norm(z, w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
