"""gated_ffn and its gradients against the formula in 64 bits.

Bounds: every output passes two roundings to the 16-bit type on its way (the product
act * up, or the gradients of both projections, as the next matrix product's
operand; and the output), each of at most the roundoff u of an element and
u / sqrt(3) in the 2-norm when errors spread evenly: sqrt(2 / 3) u, bounded by
1.25 u for small outputs."""

import pytest
import torch

from encoder_plain import ROUNDOFF, gated_ffn64, off
from late_interaction_kernels.encoder import gated_ffn

pytestmark = pytest.mark.gpu


def _case(*tag):
    print("[case]", *tag, flush=True)


def _make(rows, d, f, dtype, residual, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, d, generator=g).to(dtype)
    wi = (torch.randn(2 * f, d, generator=g) * d**-0.5).to(dtype)
    wo = (torch.randn(d, f, generator=g) * f**-0.5).to(dtype)
    r = torch.randn(rows, d, generator=g).to(dtype) if residual else None
    gy = torch.randn(rows, d, generator=g).to(dtype)
    return x, wi, wo, r, gy


def _grads64(x, wi, wo, r, gy, act):
    leaves = [t.double().requires_grad_() for t in (x, wi, wo)]
    y = gated_ffn64(*leaves, None if r is None else r.double(), act)
    return y.detach(), torch.autograd.grad(y, leaves, gy.double())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows,d,f,residual", [(1, 64, 48, True), (3, 8, 8, False), (32, 128, 200, True),
                                               (65, 72, 136, False), (257, 264, 520, True), (1000, 96, 64, True)])
def test_values_and_gradients(dtype, act, rows, d, f, residual):
    _case(dtype, act, rows, d, f, residual)
    x, wi, wo, r, gy = _make(rows, d, f, dtype, residual)
    y64, g64 = _grads64(x, wi, wo, r, gy, act)
    xs, wis, wos = (t.cuda().requires_grad_() for t in (x, wi, wo))
    rs = None if r is None else r.cuda().requires_grad_()
    y = gated_ffn(xs, wis, wos, rs, activation=act)
    with torch.no_grad():
        assert torch.equal(y, gated_ffn(xs, wis, wos, rs, activation=act))
    u = 1.25 * ROUNDOFF[dtype]
    assert off(y, y64) <= u
    grads = torch.autograd.grad(y, (xs, wis, wos) + ((rs,) if residual else ()), gy.cuda())
    for name, got, want in zip(("x", "w_in", "w_out"), grads, g64):
        assert off(got, want) <= u, name
    if residual:
        assert torch.equal(grads[3].cpu(), gy)


@pytest.mark.parametrize("rows,d,f", [(1, 8, 1000), (2, 768, 1152), (16, 768, 1152), (33, 384, 1024), (64, 1024, 520),
                                      (65, 768, 1152), (129, 264, 2816), (300, 768, 1152), (5000, 136, 264)])
def test_few_and_many_rows(rows, d, f):
    """Both sides of the rules on the number of rows."""
    _case(rows, d, f)
    x, wi, wo, r, gy = _make(rows, d, f, torch.bfloat16, True)
    y64, g64 = _grads64(x, wi, wo, r, gy, "gelu")
    xs, wis, wos = (t.cuda().requires_grad_() for t in (x, wi, wo))
    y = gated_ffn(xs, wis, wos, r.cuda())
    u = 1.25 * ROUNDOFF[torch.bfloat16]
    assert off(y, y64) <= u
    for name, got, want in zip(("x", "w_in", "w_out"), torch.autograd.grad(y, (xs, wis, wos), gy.cuda()), g64):
        assert off(got, want) <= u, name


@pytest.mark.parametrize("d,f", [(50, 36), (64, 45), (7, 16)])
def test_sizes_that_are_padded(d, f):
    x, wi, wo, r, gy = _make(37, d, f, torch.float16, True)
    y64, g64 = _grads64(x, wi, wo, r, gy, "silu")
    xs, wis, wos = (t.cuda().requires_grad_() for t in (x, wi, wo))
    y = gated_ffn(xs, wis, wos, r.cuda(), activation="silu")
    u = 1.25 * ROUNDOFF[torch.float16]
    assert off(y, y64) <= u
    for got, want in zip(torch.autograd.grad(y, (xs, wis, wos), gy.cuda()), g64):
        assert off(got, want) <= u


def test_gradient_against_differences():
    """The kernel's gradient along a direction against central differences of the formula."""
    x, wi, wo, _, gy = _make(24, 64, 96, torch.float16, False)
    xs, wis, wos = (t.cuda().requires_grad_() for t in (x, wi, wo))
    grads = torch.autograd.grad(gated_ffn(xs, wis, wos), (xs, wis, wos), gy.cuda())
    g = torch.Generator().manual_seed(5)
    for k, grad in enumerate(grads):
        v = torch.randn(grad.shape, generator=g, dtype=torch.float64)

        def f(step):
            a = [x.double(), wi.double(), wo.double()]
            a[k] = a[k] + step * v
            return (gated_ffn64(*a, None, "gelu") * gy.double()).sum()

        want = float((f(1e-5) - f(-1e-5)) / 2e-5)
        # errors of the gradient's elements are independent of v: their sum is about off(grad) |grad| |v| / sqrt(n)
        bound = 4 * ROUNDOFF[torch.float16] * float(grad.double().norm().cpu() * v.norm()) / v.numel() ** 0.5
        assert abs(float((grad.double().cpu() * v).sum()) - want) <= bound


def test_strides_leading_dims_and_order():
    x, wi, wo, r, gy = _make(300, 128, 192, torch.bfloat16, True)
    wide = torch.zeros(300, 200, dtype=torch.bfloat16)
    wide[:, 8:136] = x
    xs = wide.cuda()[:, 8:136].requires_grad_()
    wis, wos, rs = wi.cuda().requires_grad_(), wo.cuda().t().contiguous().t().requires_grad_(), r.cuda()
    y = gated_ffn(xs, wis, wos, rs)
    flat = gated_ffn(x.cuda(), wis, wo.cuda(), rs)
    assert torch.equal(y, flat)
    assert torch.equal(gated_ffn(x.cuda().view(3, 100, 128), wis, wos, rs.view(3, 100, 128)).view(300, 128), flat)
    one = torch.autograd.grad(gated_ffn(xs, wis, wos, rs), (xs, wis, wos), gy.cuda())
    two = torch.autograd.grad(gated_ffn(xs, wis, wos, rs), (xs, wis, wos), gy.cuda())
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_rows_stay_apart_and_empty_calls():
    x, wi, wo, _, gy = _make(70, 64, 64, torch.bfloat16, False)
    xs, wis, wos = x.cuda(), wi.cuda().requires_grad_(), wo.cuda().requires_grad_()
    want = gated_ffn(xs, wis, wos)
    bad = xs.clone()
    bad[3] = float("nan")
    bad[40, 5] = float("inf")
    y = gated_ffn(bad, wis, wos)
    keep = [i for i in range(70) if i not in (3, 40)]
    assert torch.equal(y[keep], want[keep]) and not torch.isfinite(y[3]).any()
    e = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = gated_ffn(e, wis, wos)
    ge, gi, go = torch.autograd.grad(y, (e, wis, wos), torch.empty_like(y))
    assert y.shape == (0, 64) and not gi.any() and not go.any()


def test_side_stream():
    x, wi, wo, r, _ = (None if t is None else t.cuda() for t in _make(500, 256, 384, torch.bfloat16, True))
    want = gated_ffn(x, wi, wo, r)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = x * 2 - x
        got = gated_ffn(z, wi, wo, r)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
