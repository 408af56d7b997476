"""The layer norm's C entry points: no success that leaves a wanted gradient unwritten, and no launch on
rows that do not start on an element."""

import pytest
import torch

from late_interaction_kernels import _lib

pytestmark = pytest.mark.gpu


def test_backward_of_no_rows_is_refused():
    lib = _lib.load()
    x = torch.randn(4, 64, device="cuda")
    gx, gw, gb = torch.empty_like(x), torch.empty(64, device="cuda"), torch.empty(64, device="cuda")
    stats, w = torch.ones(4, 2, device="cuda"), torch.ones(64, device="cuda")
    need = lib.lik_layer_norm_backward_workspace_size(_lib.LIK_F32, 4, 64)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def call(rows, w_grad, b_grad):
        return lib.lik_layer_norm_backward(x.data_ptr(), 64, None, 0, x.data_ptr(), 64, stats.data_ptr(), _lib.LIK_F32, rows, 64,
                                           w.data_ptr(), _lib.LIK_F32, gx.data_ptr(), w_grad, b_grad, ws.data_ptr(), need,
                                           _lib.stream_of(x))

    assert call(4, gw.data_ptr(), gb.data_ptr()) == _lib.LIK_OK
    assert call(0, gw.data_ptr(), None) == _lib.LIK_ERR_INVALID
    assert call(0, None, gb.data_ptr()) == _lib.LIK_ERR_INVALID
    assert call(0, None, None) == _lib.LIK_OK  # nothing is wanted and nothing written
    torch.cuda.synchronize()


@pytest.mark.parametrize("code,size", [(_lib.LIK_F32, 4), (_lib.LIK_BF16, 2)])
def test_rows_off_an_element_are_refused(code, size):
    lib = _lib.load()
    x = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    out = [torch.zeros(4096, dtype=torch.uint8, device="cuda") for _ in range(4)]
    p = x.data_ptr()

    def forward(x=p, r=None, w=p, b=p, y=out[0].data_ptr(), s=None, st=None):
        return lib.lik_layer_norm(x, 8, r, 8, code, 3, 8, w, b, _lib.LIK_F32, 1e-5, y, s, st, _lib.stream_of(out[0]))

    assert forward() == _lib.LIK_OK
    assert forward(x=p + size) == _lib.LIK_OK  # on an element: any row start will do
    off = size // 2
    sums = out[1].data_ptr()
    for kw in ({"x": p + off}, {"r": p + off, "s": sums}, {"r": p, "s": sums + off}, {"y": out[0].data_ptr() + off},
               {"w": p + 2}, {"b": p + 2}, {"st": out[2].data_ptr() + 2}):
        assert forward(**kw) == _lib.LIK_ERR_UNSUPPORTED, kw

    need = lib.lik_layer_norm_backward_workspace_size(code, 3, 8)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    st = torch.ones(3, 2, device="cuda")
    wg = torch.empty(2, 8, device="cuda")

    def backward(gy=p, gs=None, s=p, stats=st.data_ptr(), w=p, gx=out[0].data_ptr(), gw=wg[0].data_ptr(), gb=wg[1].data_ptr()):
        return lib.lik_layer_norm_backward(gy, 8, gs, 8, s, 8, stats, code, 3, 8, w, _lib.LIK_F32, gx, gw, gb, ws.data_ptr(),
                                           need, _lib.stream_of(x))

    assert backward() == _lib.LIK_OK
    for kw in ({"gy": p + off}, {"gs": p + off}, {"s": p + off}, {"stats": st.data_ptr() + 2}, {"w": p + 2},
               {"gx": out[0].data_ptr() + off}, {"gw": wg[0].data_ptr() + 2}, {"gb": wg[1].data_ptr() + 2}):
        assert backward(**kw) == _lib.LIK_ERR_UNSUPPORTED, kw
    torch.cuda.synchronize()
