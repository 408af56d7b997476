"""``linear_int8`` where a workgroup walks over many tiles: one to many steps of k a tile, ends inside the last row and
column tiles, every output type, against 64-bit products of the same integers (bounds as derived in
``test_gpu_linear_int8``: 2^-22 of the sum's and the bias's magnitudes, 2^-23 a rounding after that, half a step)."""

import pytest
import torch

from late_interaction_kernels.encoder import linear_int8, quantize_int8_per_token

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
ROWS = 66001  # 258 tiles of 256 rows: more than there are compute units


def _run(rows, k, n, ot, gated=False, res=False, bias=False):
    g = torch.Generator(device="cuda").manual_seed(k * n + rows)
    total = 2 * n if gated else n
    xq = torch.randint(-127, 128, (rows, k), generator=g, device="cuda", dtype=torch.int8)
    wq = torch.randint(-127, 128, (total, k), generator=g, device="cuda", dtype=torch.int8)
    xs = torch.rand(rows, generator=g, device="cuda") + 0.5
    ws = (torch.rand(total, generator=g, device="cuda") + 0.5) / (5000 * k**0.5)
    b = torch.randn(total, generator=g, device="cuda").to(ot) if bias else None
    r = torch.randn(rows, n, generator=g, device="cuda").to(ot) if res else None
    got = linear_int8(xq, wq, ws, b, r, x_scale=xs, gated=gated, out_dtype=ot)
    for lo in range(0, rows, 16384):
        part = slice(lo, lo + 16384)
        s = (xq[part].double() @ wq.double().t()) * xs[part].double()[:, None] * ws.double()
        mag = s.abs()
        if bias:
            s, mag = s + b.double(), mag + b.double().abs()
        tol = mag * 2.0**-22
        if gated:
            a, u = s[:, :n], s[:, n:]
            s, tol = a * u, tol[:, :n] * u.abs() + tol[:, n:] * a.abs() + (a * u).abs() * 2.0**-22
        if res:
            s = s + r[part].double()
            tol = tol + s.abs() * 2.0**-23
        tol = (tol + s.abs() * (torch.finfo(ot).eps / 2) + 2.0**-25) * (1 + 2.0**-10)
        off = (got[part].double() - s).abs()
        assert bool((off <= tol).all()), f"rows from {lo}: {int((off > tol).sum())} off, {float((off / tol).max()):.3g}"


@pytest.mark.parametrize("k", [16, 64, 80, 192, 512, 576, 640, 704, 1040])
def test_steps_of_k(k):
    _run(ROWS, k, 256, BF)


@pytest.mark.parametrize("ot", [BF, HF, FP])
@pytest.mark.parametrize("n", [192, 200, 256, 257, 384, 520])
@pytest.mark.parametrize("res,bias", [(False, True), (True, False)])
def test_widths(ot, n, res, bias):
    _run(ROWS, 144, n, ot, res=res, bias=bias)


@pytest.mark.parametrize("ot", [BF, HF, FP])
@pytest.mark.parametrize("n", [128, 133, 256, 264])
@pytest.mark.parametrize("res,bias", [(False, True), (True, True)])
def test_gated(ot, n, res, bias):
    _run(ROWS, 96, n, ot, gated=True, res=res, bias=bias)


@pytest.mark.parametrize("k", [64, 576, 1152])
@pytest.mark.parametrize("ot", [BF, FP])
def test_residual_over_many_steps(k, ot):
    _run(ROWS, k, 200, ot, res=True)


@pytest.mark.parametrize("rows,n", [(65537, 512), (4353, 4104), (70000, 1024)])
def test_several_tiles_a_workgroup(rows, n):
    _run(rows, 320, n, BF, bias=True)


def test_wide_rows_reach_past_32_bit_offsets():
    """256 output rows of 4.2 million fp32 columns are 4.3 GB: tiles address them by rows."""
    n, k, rows = 4200016, 16, 257
    xq = torch.randint(-127, 128, (rows, k), device="cuda", dtype=torch.int8)
    wq = torch.randint(-127, 128, (n, k), device="cuda", dtype=torch.int8)
    one = torch.ones(n, device="cuda")
    got = linear_int8(xq, wq, one, x_scale=one[:rows], out_dtype=FP)
    for i in (0, 1, 200, 255, 256):
        assert torch.equal(got[i].double(), wq.double() @ xq[i].double())


def test_captured_twice_and_replayed_with_eager_calls_between():
    wq, ws = quantize_int8_per_token(torch.randn(320, 200, device="cuda"))
    x, y = (torch.randn(ROWS, 200, device="cuda").to(BF) for _ in range(2))
    linear_int8(x, wq, ws)
    graphs, outs = [], []
    for t in (x, y):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(linear_int8(t, wq, ws, activation="silu"))
        graphs.append(g)
    for _ in range(3):
        x.normal_()
        y.normal_()
        for g in graphs:
            g.replay()
        want = [linear_int8(t, wq, ws, activation="silu") for t in (x, y)]
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        torch.cuda.synchronize()
