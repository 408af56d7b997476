"""Rows as 8-bit integers where several rows share a wavefront (more than 1024 of them): equal to the definition, bit for bit,
for every number of lanes and chunks a row, rows past the last whole group of them, and rows that start off 16 bytes."""

import pytest
import torch

from test_gpu_int8_tokens import _check

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("rows", [1025, 1027, 4099])
@pytest.mark.parametrize("d", [1, 3, 64, 65, 127, 128, 129, 193, 255, 257, 384, 400, 513, 768, 1000, 1024, 1025, 1600, 2500, 3500])
def test_equal_to_the_definition(dtype, rows, d):
    g = torch.Generator(device="cuda").manual_seed(rows * d)
    x = torch.randn(rows, d + 3, generator=g, device="cuda") * torch.logspace(-3, 3, rows, device="cuda")[:, None]
    x[5, d // 2], x[rows - 1, d], x[rows // 2, 0] = float("inf"), float("nan"), 1e4
    x[7], x[rows - 2] = 0.0, -0.0
    x = x.to(dtype)
    for part in (x[:, 1:d + 1], x[:, :d].contiguous()):
        _check(part)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("d", [16, 96, 200, 500])
def test_the_largest_is_found_on_every_lane(dtype, d):
    """Row r has its largest element at r % d, so each lane's and chunk's turn comes."""
    rows = 1030 + d
    x = torch.rand(rows, d, device="cuda") - 0.5
    at = torch.arange(rows, device="cuda")
    x[at, at % d] = torch.where(at % 2 == 0, 3.0, -3.0) + torch.rand(rows, device="cuda")
    q, s = _check(x.to(dtype))
    assert bool((q[at, at % d].abs() == 127).all())
