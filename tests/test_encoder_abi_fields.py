"""The packed argument structs of the rotation and the 8-bit linear layer mirror include/lik.h (no GPU needed), and what
the entry points refuse before any launch."""

import ctypes
import re
import struct
from pathlib import Path

import pytest

from late_interaction_kernels import _lib

TEXT = re.sub(r"/\*.*?\*/", "", (Path(__file__).resolve().parents[1] / "include" / "lik.h").read_text(), flags=re.S)
C = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float}


@pytest.mark.parametrize("name,cls,pack", [("lik_rotary_t", _lib.LikRotary, _lib.pack_rotary),
                                           ("lik_linear_int8_t", _lib.LikLinearInt8, _lib.pack_linear_int8)])
def test_structs_match_the_header(name, cls, pack):
    body = re.search(r"typedef struct \{([^{}]*)\}\s*" + name, TEXT).group(1)
    fields = re.findall(r"(?:const\s+)?(\w+)\s*(\*?)\s*(\w+)\s*;", body)
    want = [(n.replace("in", "in_features") if n == "in" else n, ctypes.c_void_p if star else C[t]) for t, star, n in fields]
    assert list(cls._fields_) == want
    values = [i + 1 for i in range(len(want))]
    obj = cls(*values)
    assert pack(*values) == bytes(obj)[:struct.calcsize("@" + "".join("P" if t is ctypes.c_void_p else "q" if t is ctypes.c_int64
                                                                     else "i" if t is ctypes.c_int32 else "f" for _, t in want))]


def _library():
    if not _lib.library_path().exists():
        pytest.skip("the library is not built")
    return _lib.load()


def test_statuses_before_any_launch():
    lib = _library()
    ok = dict(x=16, x_scale=0, weight=16, weight_scale=16, bias=0, residual=0, x_stride=64, weight_stride=64,
              residual_stride=0, rows=4, in_features=64, out_features=8, x_dtype=0, out_dtype=0, bias_dtype=0,
              activation=-1, gated=0)

    def call(out=16, ws=0, nbytes=0, **kw):
        return lib.lik_linear_int8(_lib.pack_linear_int8(*{**ok, **kw}.values()), out, ws, nbytes, None)

    assert lib.lik_linear_int8(None, 16, None, 0, None) == -1
    assert call(rows=0) == 0
    for bad in ({"rows": -1}, {"in_features": 0}, {"out_features": 0}, {"activation": 3}, {"activation": -2}, {"x": 0},
                {"weight": 0}, {"weight_scale": 0}, {"out": 0}, {"x_dtype": 4}):
        assert call(**bad) == -1, bad
    for bad in ({"x_dtype": 3}, {"out_dtype": 4}, {"in_features": 131072}, {"x": 17}, {"weight": 24}, {"weight_stride": 72},
                {"weight_stride": -64}, {"weight_scale": 18}, {"bias": 17}, {"bias": 16, "bias_dtype": 1},
                {"x_dtype": 4, "x_scale": 16, "x": 24}, {"x_dtype": 4, "x_scale": 16, "in_features": 60}, {"out": 17},
                {"gated": 1, "out_features": 1 << 24, "weight_stride": 4096}):
        assert call(**bad) == -2, bad
    assert call(rows=1000) == -3  # (the integers and scales need a workspace)
    size = lib.lik_linear_int8_workspace_size(_lib.pack_linear_int8(*{**ok, "rows": 1000}.values()))
    assert size >= 1000 * 64 + 4000 and call(rows=1000, ws=256, nbytes=size - 1) == -3

    rot = dict(q=16, k=0, dtype=0, heads=2, kv_heads=0, dim=8, n=1, len=4, q_stride_n=64, q_stride_l=16, q_stride_h=8,
               k_stride_n=0, k_stride_l=0, k_stride_h=0, cu_seqlens=0, positions=0, position_stride_n=0,
               position_stride_l=0, offset=0, frequencies=16, position_bits=0, frequency_bits=64, pairs=4, interleaved=0,
               inverse=0, amplitude=1.0)

    def turn(out=16, **kw):
        return lib.lik_rotary(_lib.pack_rotary(*{**rot, **kw}.values()), out, None, None)

    assert lib.lik_rotary(None, 16, None, None) == -1
    assert turn(len=0) == 0 and turn(n=0) == 0 and turn(q=0) == 0
    for bad in ({"pairs": 0}, {"pairs": 5}, {"dim": 0}, {"n": -1}, {"frequencies": 0}, {"frequency_bits": 16},
                {"positions": 16, "position_bits": 16}, {"positions": 16, "position_bits": 32, "cu_seqlens": 16}, {"out": 0}):
        assert turn(**bad) == -1, bad
    for bad in ({"dtype": 3}, {"dim": 1025}, {"q": 17}, {"out": 17}, {"frequencies": 20}, {"cu_seqlens": 18}):
        assert turn(**bad) == -2, bad

    for fn, args in ((lib.lik_quantize_int8, [16, 8, 0, 2, 8, 16, 8, 16, None]),
                     (lib.lik_dequantize_int8, [16, 8, 16, 0, 2, 8, 16, None])):
        rows = 3 if fn is lib.lik_quantize_int8 else 4
        assert fn(*args[:rows], 0, *args[rows + 1:]) == 0 and fn(*args[:rows], -1, *args[rows + 1:]) == -1
        assert fn(None, *args[1:]) == -1
    assert lib.lik_quantize_int8(16, 8, 4, 2, 8, 16, 8, 16, None) == -2
    assert lib.lik_quantize_int8(16, 8, 0, 2, 8, 16, 7, 16, None) == -1
    assert lib.lik_quantize_int8(17, 8, 0, 2, 8, 16, 8, 16, None) == -2
