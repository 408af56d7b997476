"""The rotation, the 8-bit tokens and the linear layer on them refuse to write where they read, before any launch (no GPU
needed: every call here is refused)."""

import pytest

from late_interaction_kernels import _lib

INVALID = -1


@pytest.fixture(scope="module")
def lib():
    if not _lib.library_path().exists():
        pytest.skip("the library is not built")
    return _lib.load()


@pytest.mark.parametrize("q,k,q_out,k_out", [(256, 0, 256, 0), (0, 256, 0, 256), (256, 512, 512, 1024), (256, 512, 1024, 256),
                                             (256, 512, 1024, 1024)])
def test_rotary(lib, q, k, q_out, k_out):
    a = _lib.pack_rotary(q, k, 0, 2, 2, 8, 1, 4, 64, 16, 8, 64, 16, 8, 0, 0, 0, 0, 0, 16, 0, 64, 4, 0, 0, 1.0)
    assert lib.lik_rotary(a, q_out, k_out, None) == INVALID


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_tokens(lib, dtype):
    assert lib.lik_quantize_int8(256, 8, dtype, 2, 8, 256, 8, 16, None) == INVALID
    assert lib.lik_dequantize_int8(256, 8, 16, dtype, 2, 8, 256, None) == INVALID


@pytest.mark.parametrize("out", [256, 512])
def test_linear(lib, out):
    a = _lib.pack_linear_int8(256, 16, 512, 16, 0, 0, 64, 64, 0, 4, 64, 8, 4, 0, 0, -1, 0)
    assert lib.lik_linear_int8(a, out, None, 0, None) == INVALID
