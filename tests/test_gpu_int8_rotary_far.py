"""Rotation, 8-bit tokens and linear layers on rows more than 2^32 bytes apart, on the same tensor twice, and the
rotation's forward and backward pass in one captured graph."""

import pytest
import torch

from late_interaction_kernels.encoder import (dequantize_int8_per_token, linear_int8, quantize_int8_per_token, rotary,
                                              rotary_frequencies)

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
FAR = 2**32 + 16


@pytest.fixture(scope="module")
def far():
    """Two rows of 4096 elements (viewed as bf16), FAR elements apart."""
    base = torch.empty(FAR + 4096, dtype=BF, device="cuda")
    rows = base.as_strided((2, 4096), (FAR, 1))
    rows.copy_(torch.randn(2, 4096, device="cuda"))
    yield rows
    del base, rows
    torch.cuda.empty_cache()


def test_far_rows(far):
    near = far.clone()
    f, _ = rotary_frequencies(64, device="cuda")
    for shape in ((2, 1, 4, 64), (1, 2, 4, 64), (1, 1, 2, 64)):
        strides = [FAR if n == 2 else 64 for n in shape[:3]] + [1]
        if shape[2] == 4:
            strides[2] = 64
        x = far.as_strided(shape, strides)
        y = near[:, :256].reshape(2, 4, 64)[:, :shape[2] if shape[2] == 4 else 1].reshape(shape)
        assert torch.equal(rotary(x, frequencies=f, offset=3), rotary(y, frequencies=f, offset=3))
    for d in (64, 1000, 4096):
        got, want = quantize_int8_per_token(far[:, :d]), quantize_int8_per_token(near[:, :d])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    q8 = far.view(torch.int8)[:, :777]
    scale = torch.rand(2, device="cuda")
    assert torch.equal(dequantize_int8_per_token(q8, scale), dequantize_int8_per_token(q8.clone(), scale))
    wq, ws = quantize_int8_per_token(torch.randn(48, 512, device="cuda"))
    assert torch.equal(linear_int8(far[:, :512], wq, ws, None, far[:, 512:560]),
                       linear_int8(near[:, :512], wq, ws, None, near[:, 512:560]))
    x8 = far.view(torch.int8)[:, :512]
    assert torch.equal(linear_int8(x8, wq, ws, x_scale=scale), linear_int8(x8.clone(), wq, ws, x_scale=scale))
    w2 = far.view(torch.int8)[:, 1024:1536]
    assert torch.equal(linear_int8(near[:, :512], w2, ws[:2]), linear_int8(near[:, :512], w2.clone(), ws[:2]))


def test_the_same_tensor_twice():
    f, _ = rotary_frequencies(32, device="cuda")
    x = torch.randn(2, 9, 3, 32, device="cuda", requires_grad=True)
    a, b = rotary(x, x, frequencies=f)
    assert torch.equal(a, b)
    (g,) = torch.autograd.grad((a, b), x, (torch.ones_like(a), torch.ones_like(b)))
    (h,) = torch.autograd.grad(rotary(x, frequencies=f), x, torch.ones_like(a))
    assert torch.equal(g, 2 * h)
    y = torch.randn(130, 64, device="cuda").to(BF)
    wq, ws = quantize_int8_per_token(torch.randn(64, 64, device="cuda"))
    # the residual is the input
    assert torch.equal(linear_int8(y, wq, ws, None, y), linear_int8(y, wq, ws, None, y.clone()))


def test_forward_and_backward_in_one_graph():
    f, _ = rotary_frequencies(64, device="cuda")
    x = torch.randn(1, 50, 4, 64, device="cuda").to(BF)
    w = torch.randn(1, 50, 4, 64, device="cuda").to(BF)

    def step():
        q = x.detach().requires_grad_()
        y = rotary(q, frequencies=f, interleaved=True)
        return y, torch.autograd.grad(y, q, w)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        x.normal_()
        w.normal_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        torch.cuda.synchronize()


def test_tensors_that_want_a_gradient_are_refused():
    wq, ws = quantize_int8_per_token(torch.randn(16, 32, device="cuda"))
    x = torch.randn(4, 32, device="cuda", requires_grad=True)
    bias = torch.nn.Parameter(torch.zeros(16, device="cuda"))
    for call in (lambda: quantize_int8_per_token(x), lambda: linear_int8(x, wq, ws),
                 lambda: linear_int8(x.detach(), wq, ws, bias),
                 lambda: dequantize_int8_per_token(wq, ws.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    with torch.no_grad():
        assert linear_int8(x, wq, ws, bias).shape == (4, 16)
    with pytest.raises(ValueError):
        rotary(torch.randn(1, 2, 1, 32, device="cuda"), frequencies=torch.ones(16, device="cuda", requires_grad=True))
