"""The C entry points of the encoder operators: what they refuse is a status, never a launch
or an abort, and calls with a workspace of exactly the stated size succeed."""

import ctypes

import pytest
import torch

from late_interaction_kernels import _lib
from late_interaction_kernels.attention import _args
from late_interaction_kernels.encoder import attention, gated_ffn

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _att(n=1, lq=1, lk=4096, h=2, hk=1, d=64):
    q = torch.randn(n, lq, h, d, device="cuda", dtype=BF)
    k, v = (torch.randn(n, lk, hk, d, device="cuda", dtype=BF) for _ in range(2))
    return q, k, v, _args(q, k, v, (-1, -1, 0.125, lq, lk), None, None, None, None)


def test_attention_statuses():
    lib = _lib.load()
    q, k, v, a = _att()
    out = torch.empty_like(q)
    need = lib.lik_attention_workspace_size(ctypes.byref(a))
    assert need > 0  # few rows over long keys are split
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    st = _lib.stream_of(q)

    def call(s=a, o=out.data_ptr(), w=ws.data_ptr(), n=need):
        return lib.lik_attention(None if s is None else ctypes.byref(s), o, None, None, w, n, st)

    assert call() == _lib.LIK_OK
    assert torch.equal(out, attention(q, k, v, scale=0.125))
    assert call(w=None) == _lib.LIK_ERR_WORKSPACE
    assert call(n=need - 1) == _lib.LIK_ERR_WORKSPACE
    assert call(s=None) == _lib.LIK_ERR_INVALID
    assert call(o=None) == _lib.LIK_ERR_INVALID
    assert call(o=out.data_ptr() + 2) == _lib.LIK_ERR_UNSUPPORTED
    for field, value, status in (("heads", 0, _lib.LIK_ERR_INVALID), ("kv_heads", 3, _lib.LIK_ERR_INVALID),
                                 ("scale", 0.0, _lib.LIK_ERR_INVALID), ("scale", float("nan"), _lib.LIK_ERR_INVALID),
                                 ("left", -2, _lib.LIK_ERR_INVALID), ("n", -1, _lib.LIK_ERR_INVALID),
                                 ("k", None, _lib.LIK_ERR_INVALID), ("cu_q", q.data_ptr(), _lib.LIK_ERR_INVALID),
                                 ("dim", 136, _lib.LIK_ERR_UNSUPPORTED), ("dim", 60, _lib.LIK_ERR_UNSUPPORTED),
                                 ("dtype", _lib.LIK_F32, _lib.LIK_ERR_UNSUPPORTED),
                                 ("q_stride_l", 12, _lib.LIK_ERR_UNSUPPORTED),
                                 ("v", v.data_ptr() + 8, _lib.LIK_ERR_UNSUPPORTED)):
        b = type(a).from_buffer_copy(a)
        setattr(b, field, value)
        assert call(s=b) == status, field
    b = type(a).from_buffer_copy(a)
    b.k_mask, b.k_len = k.data_ptr(), (1 << 18) + 1
    assert call(s=b) == _lib.LIK_ERR_UNSUPPORTED
    b = type(a).from_buffer_copy(a)
    b.n = 0
    assert call(s=b) == _lib.LIK_OK  # nothing to do
    torch.cuda.synchronize()


def test_attention_backward_statuses():
    lib = _lib.load()
    q, k, v, a = _att(lq=40, lk=50)
    out, low = torch.empty_like(q), torch.empty(q.shape, dtype=torch.int8, device="cuda")
    lse = torch.empty(2, 40, device="cuda")
    assert lib.lik_attention_workspace_size(ctypes.byref(a)) == 0
    st = _lib.stream_of(q)
    assert lib.lik_attention(ctypes.byref(a), out.data_ptr(), lse.data_ptr(), low.data_ptr(), None, 0, st) == _lib.LIK_OK
    g = torch.randn_like(q)
    gq, gk, gv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    need = lib.lik_attention_backward_workspace_size(ctypes.byref(a))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def call(o=out.data_ptr(), l=lse.data_ptr(), b=low.data_ptr(), g=g.data_ptr(), k=gk.data_ptr(), n=need):
        return lib.lik_attention_backward(ctypes.byref(a), o, l, b, g, 40 * 128, 128, 64, gq.data_ptr(), k,
                                          gv.data_ptr(), ws.data_ptr(), n, st)

    assert call() == _lib.LIK_OK
    for kw in ({"o": None}, {"l": None}, {"b": None}, {"g": None}, {"k": None}):
        assert call(**kw) == _lib.LIK_ERR_INVALID, kw
    assert call(n=need - 1) == _lib.LIK_ERR_WORKSPACE
    assert call(g=g.data_ptr() + 2) == _lib.LIK_ERR_UNSUPPORTED
    torch.cuda.synchronize()


def test_gated_ffn_and_layer_norm_statuses():
    lib = _lib.load()
    rows, d, f = 300, 64, 96
    x = torch.randn(rows, d, device="cuda", dtype=BF)
    wi, wo = torch.randn(2 * f, d, device="cuda", dtype=BF), torch.randn(d, f, device="cuda", dtype=BF)
    out, h = torch.empty_like(x), torch.empty(rows, f, device="cuda", dtype=BF)
    need = lib.lik_gated_ffn_workspace_size(_lib.LIK_BF16, rows, d, f)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    st = _lib.stream_of(x)

    def call(x=x.data_ptr(), t=_lib.LIK_BF16, d=d, f=f, act=0, n=need, xs=d):
        return lib.lik_gated_ffn(x, xs, t, rows, d, f, wi.data_ptr(), 64, wo.data_ptr(), 96, None, 0, act, out.data_ptr(),
                                 h.data_ptr(), None, ws.data_ptr(), n, st)

    assert call() == _lib.LIK_OK
    assert torch.equal(out, gated_ffn(x, wi, wo))
    assert call(x=None) == _lib.LIK_ERR_INVALID
    assert call(act=3) == _lib.LIK_ERR_INVALID
    assert call(t=_lib.LIK_F32) == _lib.LIK_ERR_UNSUPPORTED
    assert call(d=60) == _lib.LIK_ERR_UNSUPPORTED
    assert call(f=90) == _lib.LIK_ERR_UNSUPPORTED
    assert call(xs=63) == _lib.LIK_ERR_UNSUPPORTED
    assert call(x=x.data_ptr() + 2) == _lib.LIK_ERR_UNSUPPORTED
    assert call(n=need - 1) == _lib.LIK_ERR_WORKSPACE

    w = torch.ones(64, device="cuda")

    def norm(x=x.data_ptr(), d=64, t=_lib.LIK_BF16, wt=_lib.LIK_F32, w=w.data_ptr(), r=None):
        return lib.lik_layer_norm(x, 64, r, 64, t, rows, d, w, None, wt, 1e-5, out.data_ptr(), None, None, st)

    assert norm() == _lib.LIK_OK
    assert norm(x=None) == _lib.LIK_ERR_INVALID
    assert norm(w=None) == _lib.LIK_ERR_INVALID
    assert norm(r=x.data_ptr()) == _lib.LIK_ERR_INVALID  # a residual without room for the sum
    assert norm(d=0) == _lib.LIK_ERR_INVALID
    assert norm(d=8200) == _lib.LIK_ERR_UNSUPPORTED
    assert norm(t=_lib.LIK_FP8_E4M3) == _lib.LIK_ERR_UNSUPPORTED
    assert norm(wt=_lib.LIK_F16) == _lib.LIK_ERR_UNSUPPORTED
    torch.cuda.synchronize()


def test_graph_replays():
    """A captured attention and feed-forward block, replayed with eager work in between."""
    x = torch.randn(2, 70, 256, device="cuda", dtype=BF)
    wi, wo = torch.randn(768, 256, device="cuda", dtype=BF) * 0.06, torch.randn(256, 384, device="cuda", dtype=BF) * 0.05
    m = torch.arange(70, device="cuda")[None] < torch.tensor([70, 31], device="cuda")[:, None]

    def step():
        q = x.view(2, 70, 4, 64)
        a = attention(q, q, q, m, m).reshape(140, 256)
        return gated_ffn(a, wi, wo, a)

    want = step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for i in range(4):
        x.copy_(torch.randn_like(x))
        want = step()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), i


def test_ctypes_struct_matches_the_header():
    import re
    from pathlib import Path

    text = (Path(__file__).resolve().parents[1] / "include" / "lik.h").read_text()
    body = re.search(r"typedef struct \{([^{}]*)\}\s*lik_attention_t", text).group(1)
    assert [f[0] for f in _lib.LikAttention._fields_] == re.findall(r"(\w+)\s*;", body)
