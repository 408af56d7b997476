"""``linear_int8`` where the product of a token's and a channel's scale leaves fp32's range and the result does not
(bounds as derived in ``test_gpu_linear_int8``: three roundings of the scaled sum, as if nothing under- or overflowed)."""

import pytest
import torch

from late_interaction_kernels.encoder import linear_int8, quantize_int8_per_token
from test_gpu_linear_int8 import _check, _pass

pytestmark = pytest.mark.gpu
BF, HF, FP, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8
# few rows; tiles of 128 x 64 (gated: 64 x 128), 256 x 128, and walked ones of 256 x 256 and 256 x 192
SIZES = [(5, 208, 40), (33, 208, 40), (70, 208, 65), (16481, 80, 513), (66001, 80, 256), (66001, 80, 192)]


def _integers(rows, k):
    return torch.randint(-127, 128, (rows, k), device="cuda", dtype=I8)


def _cycle(n, *values):
    return torch.tensor(values, dtype=FP, device="cuda").repeat(-(-n // len(values)))[:n]


@pytest.mark.parametrize("rows,k,n", SIZES)
@pytest.mark.parametrize("ot", [BF, FP])
@pytest.mark.parametrize("xs,ws", [((1e-24, 3e-24), (1e-17, 7e-18)), ((1e36, 0.01, -2e36), (1e-34, 3e-35)),
                                   ((2.0**96, 2.0**97), (2.0**-100, 2.0**-99)), ((1e-35,), (1e30, 1.0)),
                                   ((2.0**-130, 1.0), (2.0**20, 1.0))])
def test_products_outside_the_range(rows, k, n, ot, xs, ws):
    xq, wq, xs, ws = _integers(rows, k), _integers(n, k), _cycle(rows, *xs), _cycle(n, *ws)
    _check(linear_int8(xq, wq, ws, x_scale=xs, out_dtype=ot), xq, xs, wq, ws)


@pytest.mark.parametrize("rows,k,n", SIZES)
@pytest.mark.parametrize("ot", [BF, HF, FP])
@pytest.mark.parametrize("xs,ws", [(1e25, 1e20), (1e20, 1e25), (3e36, 3e38)])
def test_sums_of_zero_stay_zero(rows, k, n, ot, xs, ws):
    xq, wq = _integers(rows, k), _integers(n, k)
    xq[:, ::2] = 0
    wq[:, 1::2] = 0
    b = torch.randn(n, device="cuda").to(ot)
    got = linear_int8(xq, wq, torch.full((n,), ws, device="cuda"), b, x_scale=torch.full((rows,), xs, device="cuda"),
                      out_dtype=ot)
    assert torch.equal(got, b.expand(rows, n))


@pytest.mark.parametrize("rows,k,n", SIZES)
@pytest.mark.parametrize("xs,ws", [((1e-24,), (1e-17, 1e20)), ((1e36, 1e35), (1e-36, 2e-36))])
def test_gated(rows, k, n, xs, ws):
    xq, wq, xs = _integers(rows, k), _integers(2 * n, k), _cycle(rows, *xs)
    ws = torch.tensor(ws, device="cuda").repeat_interleave(n)  # the gate's, the up half's
    got = linear_int8(xq, wq, ws, x_scale=xs, gated=True, out_dtype=FP).double().cpu()
    v, tol = _pass(xq.cpu(), xs.cpu(), wq.cpu(), ws.cpu(), None)
    # a half that is under 2^-126 itself is a multiple of 2^-149, so up to 2^-150 from what it rounds (a gate of 99 * 1e-41
    # has 20 bits), and that times the other half is in the product
    tol = tol + 2.0**-150
    (a, u), (ta, tu) = v.chunk(2, 1), tol.chunk(2, 1)
    want = a * u
    tol = ta * u.abs() + tu * a.abs() + ta * tu + want.abs() * (2.0**-23 + 2.0**-24) + 2.0**-149
    off = (got - want).abs() / (tol * (1 + 2.0**-10))
    assert float(off.max()) <= 1.0, f"{int((off > 1).sum())} of {off.numel()} off, worst {float(off.max()):.3f}"


@pytest.mark.parametrize("rows,k,n", SIZES[:5])
@pytest.mark.parametrize("xt,size,ws", [(FP, 1e-22, 1e-18), (FP, 1e37, 1e-36), (BF, 1e-22, 1e-18), (BF, 1e37, 1e-36)])
def test_rows_quantised_within_the_call(rows, k, n, xt, size, ws):
    x = (torch.randn(rows, k, device="cuda") * size).to(xt)
    x[1::3] = torch.randn_like(x[1::3])
    wq, ws = _integers(n, k), torch.full((n,), ws, device="cuda")
    _check(linear_int8(x, wq, ws), *quantize_int8_per_token(x), wq, ws)
