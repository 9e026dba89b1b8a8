"""What the operators along a sequence refuse, without a GPU: every check happens before the first CUDA call."""
import ctypes as C

import numpy as np
import pytest

import recpulse_b200 as rpb

BUF = np.zeros(1 << 16, np.uint8)


def at(offset=0):
    return C.c_void_p(BUF.ctypes.data + offset)


def conv(batch=2, length=5, channels=8, width=4, activation=1, **over):
    c = rpb.RpbCausalConv()
    rpb.load().rpb_causal_conv_packed(C.byref(c), batch, length, channels, width, activation)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def test_packed_convolution_geometry():
    c = conv()
    assert (c.batch, c.len, c.channels, c.width, c.activation) == (2, 5, 8, 4, 1)
    assert (c.x_batch, c.x_row, c.y_batch, c.y_row, c.dx_batch, c.dx_row) == (40, 8) * 3


@pytest.mark.parametrize("wrong", [dict(batch=0), dict(length=0), dict(length=-1), dict(channels=0), dict(width=0), dict(width=9),
                                   dict(activation=2), dict(x_row=7), dict(y_row=7), dict(y_batch=39), dict(x_batch=-40), dict(y_batch=0)])
def test_convolution_refuses_bad_geometry(wrong):
    lib = rpb.load()
    c = conv(**wrong)
    assert lib.rp_causal_conv_ex(at(0), None, at(8192), at(16384), None, None, None, C.byref(c), 0, 0, None) == -1
    if not set(wrong) <= {"x_row", "y_row", "x_batch", "y_batch"}:
        assert lib.rp_causal_conv_ws_bytes(C.byref(c), 0) == -1


def test_convolution_refuses_bad_calls():
    lib = rpb.load()
    c = conv()
    y, x, w = at(0), at(8192), at(16384)
    call = lambda *a, dtype=0, device=0: lib.rp_causal_conv_ex(*a, None, None, None, C.byref(c), dtype, device, None)      # noqa: E731
    assert call(None, None, x, w) == -1 and call(y, None, None, w) == -1 and call(y, None, x, None) == -1
    assert call(y, None, x, w, device=-1) == -1                    # host memory
    assert call(y, None, x, w, dtype=9) == -1 and call(y, None, x, w, dtype=-1) == -1
    assert call(x, None, x, w) == -1 and call(at(8192 + 4), None, x, w) == -1         # y over x
    assert lib.rp_causal_conv_ex(y, None, x, w, None, None, None, None, 0, 0, None) == -1
    grad = lambda dx, dw, ds, ws, dy, xx: lib.rp_causal_conv_grad_ex(dx, dw, None, ds, 0, dy, at(20000), xx, w, None, None, None, ws,   # noqa: E731
                                                                    C.byref(c), 0, 0, None)
    assert grad(None, None, None, None, y, x) == -1                # nothing wanted
    assert grad(None, at(30000), None, None, y, x) == -1           # filter gradient without a workspace
    assert grad(at(30000), None, None, None, None, x) == -1
    assert grad(x, None, None, None, y, x) == -1 and grad(y, None, None, None, y, x) == -1       # dx over x, over dy
    assert grad(at(30000), None, at(20000), None, y, x) == -1      # dstate_in over dstate_out
    assert lib.rp_causal_conv_ws_bytes(None, 0) == -1 and lib.rp_causal_conv_ws_bytes(C.byref(c), 7) == -1
    assert lib.rp_causal_conv_ws_bytes(C.byref(c), 0) > 0
