"""``linear_int8`` at the largest numbers of input features, which are no multiple of 16: sums stay exact up to 131071 products
of 2^14 (2^31 - 2^14), for integers and for rows quantised within the call."""

import pytest
import torch

from late_interaction_kernels import _lib
from late_interaction_kernels.encoder import linear_int8, quantize_int8_per_token

FP, I8 = torch.float32, torch.int8


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 40, 129])
@pytest.mark.parametrize("k", [131057, 131070, 131071])
def test_integers(rows, k):
    x, w = torch.full((rows, k), -128, dtype=I8, device="cuda"), torch.full((2, k), -128, dtype=I8, device="cuda")
    w[1] = 127
    got = linear_int8(x, w, torch.ones(2, device="cuda"), x_scale=torch.ones(rows, device="cuda"), out_dtype=FP)
    want = torch.tensor([16384.0 * k, -16256.0 * k], dtype=torch.float64)
    # the sum's conversion to fp32 is the only rounding
    assert bool(((got.double().cpu() - want).abs() <= want.abs() * 2.0**-24).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 129])
def test_quantised_within(rows):
    k = 131071
    x = torch.randn(rows, k, device="cuda").to(torch.bfloat16)
    wq, ws = quantize_int8_per_token(torch.randn(3, k, device="cuda"))
    xq, xs = quantize_int8_per_token(x)
    got = linear_int8(x, wq, ws, out_dtype=FP)
    assert torch.equal(got, linear_int8(xq, wq, ws, x_scale=xs, out_dtype=FP))
    want = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()
    assert bool(((got.double() - want).abs() <= want.abs() * 2.0**-22).all())


def test_statuses():
    """(no GPU needed: no rows, so no launch)"""
    if not _lib.library_path().exists():
        pytest.skip("the library is not built")
    lib = _lib.load()

    def call(width, int8):
        a = _lib.pack_linear_int8(16, 16 if int8 else 0, 16, 16, 0, 0, width, width, 0, 0, width, 8, 4 if int8 else 0, 0, 0, -1, 0)
        return lib.lik_linear_int8(a, 16, None, 0, None)

    assert call(131072, True) == 0 and call(131088, True) == -2
    assert call(131071, False) == 0 and call(131072, False) == -2
