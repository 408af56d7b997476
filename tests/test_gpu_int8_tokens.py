"""Rows as 8-bit integers: equal to the definition, bit for bit.

scale = max(fp32(max|x| / 127), 2^-126) and q = round(x / scale), ties to even. Both are
taken in 64 bits here: quotients of 24-bit numbers that are not half-integers keep 2^-33 away
from them, so rounding to 53 bits moves none across."""

import pytest
import torch

from late_interaction_kernels.encoder import dequantize_int8_per_token, quantize_int8_per_token

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _want(x):
    x = x.double().cpu()
    amax = x.abs().amax(-1)
    scale = (amax / 127).float().clamp_min(2.0**-126)
    q = torch.round(x / scale.double()[..., None])
    bad = ~torch.isfinite(x).all(-1)
    return q.masked_fill(bad[..., None], 0).to(torch.int8), scale.masked_fill(bad, float("nan"))


def _check(x):
    q, s = quantize_int8_per_token(x)
    wq, ws = _want(x)
    assert q.shape == x.shape and q.dtype == torch.int8 and s.shape == x.shape[:-1] and s.dtype == FP
    assert torch.equal(s.cpu().nan_to_num(-1.0), ws.nan_to_num(-1.0))
    assert torch.equal(q.cpu(), wq), f"{int((q.cpu() != wq).sum())} of {wq.numel()}"
    return q, s


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 7), (5, 16), (33, 96), (67, 128), (9, 129), (4, 255), (17, 768), (3, 1000),
                                    (5, 1027), (2, 1536), (7, 2049), (3, 4096), (2, 4100), (2, 20011), (0, 64)])
def test_equal_to_the_definition(dtype, rows, d):
    x = (torch.randn(rows, d, device="cuda") * torch.logspace(-3, 3, max(rows, 1), device="cuda")[:rows, None]).to(dtype)
    _check(x)


def test_many_rows():
    _check(torch.randn(200001, 16, device="cuda").to(BF))


def test_ties_and_neighbours():
    n = torch.arange(-127, 127, device="cuda").float() + 0.5
    rows = []
    for amax in (127.0, 127.0 * 2**-20, 1.0, 3.0, 0.1, 123.456, 2.0**-100, 1e30, 99.99999, 127.00001):
        s = torch.tensor(amax, device="cuda") / 127
        mid = n * s
        up, down = torch.nextafter(mid, mid + s), torch.nextafter(mid, mid - s)
        rows.append(torch.cat([torch.tensor([amax], device="cuda"), mid, up, down, -mid[:100]]).clamp(-amax, amax))
    x = torch.stack(rows)
    for dtype in (FP, BF, HF):
        _check(x.to(dtype) if dtype != HF else x[:7].to(HF))


def test_rows_of_zeros_and_smallest_values():
    x = torch.zeros(6, 40, device="cuda")
    x[1, 3], x[2] = -0.0, 2.0**-149
    x[3, :5] = torch.tensor([2.0**-126, -(2.0**-127), 2.0**-128, 3 * 2.0**-149, 127 * 2.0**-127])
    x[4, 0], x[5, 0] = 3.4028234e38, -1e-20
    q, s = _check(x)
    assert not q[:2].any() and bool((s[:2] == 2.0**-126).all())
    _check(torch.tensor([[2.0**-24, -(2.0**-23), 0.0, 65504.0], [2.0**-24, 0, 0, 0]], device="cuda").to(HF))


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_rows_that_are_not_finite(dtype):
    x = torch.randn(6, 200, device="cuda").to(dtype)
    x[1, 7], x[3, 199], x[4, 0] = float("inf"), float("nan"), -float("inf")
    q, s = _check(x)
    assert s.isnan().tolist() == [False, True, False, True, True, False]
    back = dequantize_int8_per_token(q, s, dtype)
    assert back[1].isnan().all() and back[3].isnan().all() and torch.isfinite(back[5]).all()


def test_strides_and_shapes():
    base = torch.randn(6, 5, 70, device="cuda").to(BF)
    for x in (base, base[:, 1:4, 3:68], base.transpose(0, 1), base[..., ::2], base.permute(2, 0, 1), base[0, 0],
              base[:, :1].expand(6, 9, 70)):
        _check(x)
    assert quantize_int8_per_token(torch.zeros(3, 0, 8, device="cuda"))[1].shape == (3, 0)


@pytest.mark.parametrize("out", [BF, HF, FP])
@pytest.mark.parametrize("rows,d", [(1, 1), (7, 15), (5, 16), (33, 128), (3, 257), (2, 5000), (0, 9)])
def test_back(out, rows, d):
    q = torch.randint(-128, 128, (rows, d + 3), device="cuda", dtype=torch.int8)[:, 2:d + 2]
    s = torch.rand(rows, 2, device="cuda")[:, 1]
    got = dequantize_int8_per_token(q, s, out)
    want = (q.double() * s.double()[:, None]).float().to(out) if out == FP else None
    assert got.shape == q.shape and got.dtype == out
    if out == FP:
        assert torch.equal(got, want)
    else:  # rounded to fp32, then once more: half a step and 2^-24
        exact = q.double() * s.double()[:, None]
        tol = exact.abs() * (torch.finfo(out).eps / 2 + 2.0**-24) * (1 + 2.0**-7) + 2.0**-25
        assert bool(((got.double() - exact).abs() <= tol).all())


def test_round_trip_keeps_half_a_step():
    x = torch.randn(50, 333, device="cuda")
    q, s = quantize_int8_per_token(x)
    err = (dequantize_int8_per_token(q, s) - x).abs()
    assert bool((err <= s[:, None] * (0.5 + 127 * 2.0**-23)).all())


def test_other_stream_and_graph():
    x = torch.randn(40, 768, device="cuda").to(BF)
    want = quantize_int8_per_token(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = quantize_int8_per_token(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, s = quantize_int8_per_token(x)
        y = dequantize_int8_per_token(q, s, BF)
    for _ in range(3):
        x.normal_()
        graph.replay()
        wq, ws = quantize_int8_per_token(x)
        assert torch.equal(q, wq) and torch.equal(s, ws) and torch.equal(y, dequantize_int8_per_token(wq, ws, BF))


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("d", [4095, 4097, 6001, 8191, 8193, 16383, 16385])
def test_wide_rows(dtype, d):
    q, s = _check(torch.randn(5, d + 3, device="cuda").to(dtype)[:, 1:d + 1])
    assert torch.equal(dequantize_int8_per_token(q, s), q.float() * s[:, None])
