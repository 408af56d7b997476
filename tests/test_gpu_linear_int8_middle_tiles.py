"""``linear_int8`` where tiles of 256 x 128 fill the compute units and those of 256 x 256 do not (16480 rows to 768 features): fewer
and more steps of k than there are stages, ends inside the last row and column tiles, every output type and epilogue (bounds as in
``test_gpu_linear_int8``). The integers are those of the definition in 64 bits."""

import pytest
import torch

from late_interaction_kernels.encoder import linear_int8
from test_gpu_int8_tokens import _want
from test_gpu_linear_int8 import _check
from test_gpu_linear_int8_tiles import _run

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
SIZES = [(16481, 768), (20001, 513), (33000, 130), (32769, 256)]


@pytest.mark.parametrize("rows,n", SIZES)
@pytest.mark.parametrize("k", [16, 80, 192, 1040])
@pytest.mark.parametrize("ot", [BF, HF, FP])
@pytest.mark.parametrize("res,bias", [(False, False), (True, True)])
def test_sums(rows, n, k, ot, res, bias):
    _run(rows, k, n, ot, res=res, bias=bias)


@pytest.mark.parametrize("rows,n", SIZES[:2])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("ot", [BF, HF, FP])
def test_rows_quantised_within_the_call(rows, n, act, ot):
    x = (2 * torch.randn(rows, 203, device="cuda")).to(ot)
    wq, ws = (t.cuda() for t in _want(torch.randn(n, 203) * 0.07))
    bias, r = torch.randn(n, device="cuda"), torch.randn(rows, n, device="cuda").to(ot)
    _check(linear_int8(x, wq, ws, bias, r, activation=act), *_want(x), wq, ws, bias, r, act)


@pytest.mark.parametrize("rows,k", [(1025, 130), (1500, 384), (5000, 768)])
@pytest.mark.parametrize("xt", [BF, HF, FP])
def test_integers_are_the_definitions(rows, k, xt):
    """Rows quantised many to a wavefront."""
    x = torch.randn(rows, k, device="cuda").to(xt)
    wq, ws = (t.cuda() for t in _want(torch.randn(96, k) * k**-0.5))
    _check(linear_int8(x, wq, ws), *_want(x), wq, ws)


@pytest.mark.parametrize("k", [512, 528])
@pytest.mark.parametrize("ot", [BF, FP])
def test_both_sides_of_the_width_of_walked_tiles(k, ot):
    """4 rounds of 256 columns or 5 of 192, by the number of steps."""
    _run(65793, k, 768, ot, bias=True)
