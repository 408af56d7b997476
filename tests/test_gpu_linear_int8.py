"""``linear_int8`` against its definition in 64 bits.

The integers are those of ``quantize_int8_per_token`` (held to its definition bit for bit
elsewhere), their sums are exact, so what is off comes after: three fp32 roundings of the scaled
sum (converted, times the scales, plus the bias): 2^-22 (|sum| + |bias|); the activation's own
error; one rounding of the product and one of the residual's sum, 2^-23 each; half a step of the output's type.
Activations: the erf of gelu is off by 1.5e-7, so x cdf by 1e-7 |x|; exponentials of an
argument z are off by 2^-23 (|z| + 2) of themselves, and so are the sigmoids made of them, twice that with the reciprocal."""

import math

import pytest
import torch

from encoder_plain import act64, off
from late_interaction_kernels.encoder import (attention_varlen, dequantize_int8_per_token, layer_norm, linear_int8,
                                              quantize_int8_per_token, rotary, rotary_frequencies)

pytestmark = pytest.mark.gpu
BF, HF, FP, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8
SMALLEST = {BF: 2.0**-133, HF: 2.0**-24, FP: 2.0**-149}


def _pass(xq, xs, wq, ws, b):
    """v, and how far fp32 may be from it."""
    s = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()
    bias = torch.zeros(ws.shape[0], dtype=torch.float64) if b is None else b.double()
    return s + bias, (s.abs() + bias.abs()) * 2.0**-22


def _act(v, tol, name):
    if name is None:
        return v, tol
    a = act64(v, name)
    if name == "gelu":
        own = v.abs() * 1e-7 + a.abs() * 2.0**-21
    else:
        z = v.abs() if name == "silu" else 1.6 * (v * (1 + 0.0448 * v * v)).abs().clamp(max=64.0)
        own = a.abs() * (z + 4) * 2.0**-22 + 2.0**-100
    return a, 1.2 * tol + own  # (slopes up to 1.13)


def _check(got, xq, xs, wq, ws, b=None, r=None, act=None, gated=False):
    xq, xs, wq, ws, b, r = (None if t is None else t.cpu() for t in (xq, xs, wq, ws, b, r))
    v, tol = _pass(xq.reshape(-1, xq.shape[-1]), xs.reshape(-1), wq, ws, b)
    if gated:
        n = wq.shape[0] // 2
        a, ta = _act(v[:, :n], tol[:, :n], act)
        want, tol = a * v[:, n:], ta * v[:, n:].abs() + tol[:, n:] * a.abs() + ta * tol[:, n:]
    else:
        want, tol = _act(v, tol, act)
    tol = tol + want.abs() * 2.0**-23
    if r is not None:
        r = r.double().reshape(want.shape)
        want = want + r
        tol = tol + want.abs() * 2.0**-23
    g = got.double().cpu().reshape(want.shape)
    tol = (tol + want.abs() * torch.finfo(got.dtype).eps / 2 + SMALLEST[got.dtype]) * (1 + 2.0**-10)
    bad = (g - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((g - want).abs() / tol).max()):.3f}"


def _weight(n, k):
    return quantize_int8_per_token(torch.randn(n, k, device="cuda") * k**-0.5)


ROWS = [1, 2, 31, 32, 33, 64, 65, 130, 300]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("k,n", [(64, 64), (768, 96), (16, 33), (1040, 257), (3, 5), (77, 130), (1, 1), (4096, 40),
                                 (2005, 72)])
@pytest.mark.parametrize("xt,ot", [(BF, BF), (HF, HF), (FP, FP), (I8, BF), (I8, FP), (BF, HF)])
def test_rows_and_sizes(rows, k, n, xt, ot):
    x = torch.randn(rows, k, device="cuda")
    wq, ws = _weight(n, k)
    if xt == I8:
        xq, xs = quantize_int8_per_token(x)
        _check(linear_int8(xq, wq, ws, x_scale=xs, out_dtype=ot), xq, xs, wq, ws)
    else:
        x = x.to(xt)
        _check(linear_int8(x, wq, ws, out_dtype=ot), *quantize_int8_per_token(x), wq, ws)


@pytest.mark.parametrize("rows", [3, 50, 200, 1100])
@pytest.mark.parametrize("act", [None, "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("ot", [BF, HF, FP])
@pytest.mark.parametrize("n", [128, 45])
def test_epilogues(rows, act, gated, ot, n):
    k, total = 160, 2 * n if gated else n
    x = (2 * torch.randn(rows, k, device="cuda")).to(ot)
    wq, ws = _weight(total, k)
    xq, xs = quantize_int8_per_token(x)
    for bias in (None, torch.randn(total, device="cuda").to(ot), torch.randn(total, device="cuda")):
        for r in (None, torch.randn(rows, n, device="cuda").to(ot)):
            _check(linear_int8(x, wq, ws, bias, r, activation=act, gated=gated), xq, xs, wq, ws, bias, r, act, gated)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,k,n", [(5000, 768, 1000), (2049, 1152, 768), (9001, 320, 513)])
def test_many_rows(rows, k, n, gated):
    """More tiles than compute units, ends inside tiles."""
    x = torch.randn(rows, k, device="cuda").to(BF)
    wq, ws = _weight(2 * n if gated else n, k)
    r = torch.randn(rows, n, device="cuda").to(BF)
    got = linear_int8(x, wq, ws, None, r, activation="silu", gated=gated)
    _check(got, *quantize_int8_per_token(x), wq, ws, None, r, "silu", gated)


@pytest.mark.parametrize("rows", [4, 40, 129, 3000])
def test_sums_are_exact_at_the_largest_magnitudes(rows):
    """Integers of -128 and 127 over the longest rows: sums of 2^31 - 2^14, and one off each way."""
    k = 131056  # a multiple of 16 (the kernels' own bound is 131071)
    x = torch.full((rows, k), -128, dtype=I8, device="cuda")
    w = torch.full((3, k), -128, dtype=I8, device="cuda")
    w[1] = 127
    w[2, 0] = -127
    one = torch.ones(rows, device="cuda")
    got = linear_int8(x, w, torch.ones(3, device="cuda"), x_scale=one, out_dtype=FP).double().cpu()
    want = torch.tensor([16384.0 * k, -16256.0 * k, 16384.0 * k - 128]).expand(rows, 3)
    assert bool(((got - want).abs() <= want.abs() * 2.0**-22).all())
    # differences of sums: large terms that cancel leave the exact small one
    x[:, ::2] = 127
    x[:, 1::2] = -127
    x[:, 5] = 3
    got = linear_int8(x, torch.full((1, k), 127, dtype=I8, device="cuda"), torch.ones(1, device="cuda"), x_scale=one,
                      out_dtype=FP)
    assert torch.equal(got, torch.full_like(got, 127.0 * 130))


def test_rows_that_are_not_finite_and_empty_ones():
    for rows in (6, 70, 300):
        x = torch.randn(rows, 96, device="cuda").to(HF)
        x[1, 5], x[3, 90], x[4] = float("inf"), float("nan"), 0.0
        wq, ws = _weight(40, 96)
        b = torch.randn(40, device="cuda").to(HF)
        for act in (None, "gelu", "gelu_tanh", "silu"):
            y = linear_int8(x, wq, ws, b, activation=act)
            assert y[1].isnan().all() and y[3].isnan().all()
            keep = [i for i in range(rows) if i not in (1, 3)]
            _check(y[keep], *quantize_int8_per_token(x[keep]), wq, ws, b, None, act)
    wq, ws = _weight(8, 32)
    for shape in ((0, 32), (3, 0, 32)):
        assert linear_int8(torch.zeros(*shape, device="cuda"), wq, ws).shape == (*shape[:-1], 8)


@pytest.mark.parametrize("rows", [20, 500])
def test_strides_and_shapes(rows):
    k, n = 96, 72
    wide = torch.randint(-127, 128, (n, 128), dtype=I8, device="cuda")
    ws = torch.rand(2 * n, device="cuda")[::2]
    base = torch.randn(rows, 3, 140, device="cuda").to(BF)
    r = torch.randn(rows, 3, 2 * n, device="cuda").to(BF)[..., n - 1:2 * n - 1]
    bias = torch.randn(2 * n, device="cuda").to(BF)[1::2]
    for x in (base[..., 7:7 + k], base[:, 1:2, :k].expand(rows, 3, k), base[..., :2 * 70:2][..., :k // 2].repeat(1, 1, 2)):
        xq, xs = quantize_int8_per_token(x)
        for w in (wide[:, :k], wide[:, 16:112], wide[:, 5:5 + k], wide.t().contiguous().t()[:, :k]):
            got = linear_int8(x, w, ws, bias, r)
            assert got.shape == r.shape and got.is_contiguous()
            _check(got, xq, xs, w, ws, bias, r)
            assert torch.equal(linear_int8(xq, w, ws, bias, r, x_scale=xs), got)
            assert torch.equal(linear_int8(xq.transpose(0, 1).contiguous().transpose(0, 1), w, ws, bias, r, x_scale=xs), got)
    for kk in (90, 95):  # widths that are no multiple of 16, in wider storage and at its end
        xq, xs = quantize_int8_per_token(base[:, 0, :kk])
        for w in (wide[:, :kk], wide[:, 112:][:, :16].reshape(-1)[:n * 16].view(n, 16)[:, :kk % 16 or 16]):
            x = base[:, 0, :w.shape[1]]
            xq, xs = quantize_int8_per_token(x)
            _check(linear_int8(x, w, ws), xq, xs, w, ws)
            _check(linear_int8(xq, w, ws, x_scale=xs), xq, xs, w, ws)
    one = torch.randn(k, device="cuda").to(BF)
    _check(linear_int8(one, wide[:, :k], ws)[None], *(t[None] for t in quantize_int8_per_token(one)), wide[:, :k], ws)


def test_other_stream_graph_and_two_at_once():
    k, n = 128, 256
    wq, ws = _weight(n, k)
    for rows in (16, 700, 9000):
        x = torch.randn(rows, k, device="cuda").to(BF)
        want = linear_int8(x, wq, ws, activation="gelu")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a = [linear_int8(x, wq, ws, activation="gelu") for _ in range(4)]
        b = [linear_int8(x, wq, ws, activation="gelu") for _ in range(4)]
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(want, y) for y in a + b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = linear_int8(x, wq, ws, activation="gelu")
        for _ in range(3):
            x.normal_()
            graph.replay()
            assert torch.equal(y, linear_int8(x, wq, ws, activation="gelu"))
            torch.cuda.synchronize()


def _exact_linear(x, w, b=None):
    y = x @ w.t()
    return y if b is None else y + b


def test_a_layer_in_8_bits():
    """Norm, projection, rotation, attention, projection back and a gated block, next to the same layer on the
    weights' own values in 64 bits with nothing quantised but them."""
    torch.manual_seed(5)
    d, h, hk, dh, f = 256, 4, 2, 64, 384
    cu = torch.tensor([0, 37, 120, 121], dtype=torch.int32, device="cuda")
    s = torch.randn(121, d, device="cuda").to(BF)
    norm = torch.ones(d, device="cuda")
    ws = {"qkv": _weight((h + 2 * hk) * dh, d), "o": _weight(d, h * dh), "in": _weight(2 * f, d), "out": _weight(d, f)}
    fr, _ = rotary_frequencies(dh, device="cuda")
    y = layer_norm(s, norm)
    q, k, v = linear_int8(y, *ws["qkv"]).view(-1, h + 2 * hk, dh).split([h, hk, hk], 1)
    q, k = rotary(q, k, frequencies=fr, cu_seqlens=cu)
    a = attention_varlen(q, k, v, cu, cu, 83, 83)
    s1 = linear_int8(a.flatten(1), *ws["o"], residual=s)
    got = linear_int8(linear_int8(layer_norm(s1, norm), *ws["in"], activation="silu", gated=True), *ws["out"], residual=s1)

    w = {n: (i.double() * sc.double()[:, None]).cpu() for n, (i, sc) in ws.items()}

    def ln(x):
        return torch.nn.functional.layer_norm(x, (d,))

    x = s.double().cpu()
    q, k, v = _exact_linear(ln(x), w["qkv"]).view(-1, h + 2 * hk, dh).split([h, hk, hk], 1)
    outs = []
    for lo, hi in zip(cu.tolist(), cu.tolist()[1:]):
        t = torch.arange(hi - lo, dtype=torch.float64)[:, None] * fr.cpu()
        c, sn = torch.cos(t)[:, None], torch.sin(t)[:, None]

        def turn(z):
            z1, z2 = z.chunk(2, -1)
            return torch.cat([z1 * c - z2 * sn, z2 * c + z1 * sn], -1)

        qq, kk, vv = turn(q[lo:hi]), turn(k[lo:hi]).repeat_interleave(2, 1), v[lo:hi].repeat_interleave(2, 1)
        p = torch.softmax(torch.einsum("ihd,jhd->hij", qq, kk) / math.sqrt(dh), -1)
        outs.append(torch.einsum("hij,jhd->ihd", p, vv))
    x = x + _exact_linear(torch.cat(outs).flatten(1), w["o"])
    g, u = _exact_linear(ln(x), w["in"]).chunk(2, -1)
    x = x + _exact_linear(torch.nn.functional.silu(g) * u, w["out"])
    # a token's integers are off by up to half a step of max / 127, 0.3 steps of about 3.5 / 127 in the mean: 0.8% of each
    # product's terms; four products in a row, none of which dominates the residual's sum, and bf16's 0.4% a rounding
    assert off(got, x) <= 0.03


def test_quantising_first_or_within_is_one():
    x = torch.randn(333, 200, device="cuda").to(HF)
    wq, ws = _weight(64, 200)
    xq, xs = quantize_int8_per_token(x)
    for rows in (1, 32, 64, 333):
        assert torch.equal(linear_int8(x[:rows], wq, ws), linear_int8(xq[:rows], wq, ws, x_scale=xs[:rows], out_dtype=HF))
    back = dequantize_int8_per_token(xq, xs).double() @ dequantize_int8_per_token(wq, ws).double().t()
    assert off(linear_int8(x, wq, ws), back) <= 2.0**-11
