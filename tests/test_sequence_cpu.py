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
                                   dict(activation=2), dict(batch=(1 << 30) + 1), dict(length=(1 << 30) + 1), dict(channels=(1 << 24) + 1), dict(x_row=7), dict(y_row=7), dict(y_batch=39), dict(x_batch=-40), dict(y_batch=0)])
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


def scan(batch=2, length=5, channels=8, states=4, groups=2, softplus=1, **over):
    c = rpb.RpbScan()
    rpb.load().rpb_scan_packed(C.byref(c), batch, length, channels, states, groups, softplus)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def test_packed_scan_geometry_and_sizes():
    lib, c = rpb.load(), scan()
    assert (c.x_batch, c.x_row, c.b_batch, c.b_row, c.dz_batch, c.dz_row) == (40, 8, 40, 8, 40, 8)
    assert lib.rp_selective_scan_saved_elems(C.byref(c), 0) == 2 * 1 * 8 * 4
    assert lib.rp_selective_scan_saved_elems(C.byref(scan(length=9)), 0) == 2 * 2 * 8 * 4
    assert lib.rp_selective_scan_ws_bytes(C.byref(c), 0, 0) == 0 and lib.rp_selective_scan_ws_bytes(C.byref(c), 0, 1) > 0
    assert lib.rp_selective_scan_ws_bytes(C.byref(scan(batch=1, length=4096)), 0, 0) > 0         # few channels, long: split


@pytest.mark.parametrize("wrong", [dict(batch=0), dict(length=0), dict(channels=0), dict(states=0), dict(states=65), dict(groups=0), dict(groups=3),
                                   dict(softplus=2), dict(batch=(1 << 30) + 1), dict(length=(1 << 30) + 1), dict(channels=(1 << 24) + 2), dict(x_row=7), dict(dt_row=1), dict(b_row=7), dict(c_row=7), dict(z_row=7), dict(y_row=7),
                                   dict(y_batch=39), dict(x_batch=-1)])
def test_scan_refuses_bad_geometry(wrong):
    lib, c = rpb.load(), scan(**wrong)
    a = [at(2048 * i) for i in range(9)]
    assert lib.rp_selective_scan_ex(a[0], None, None, a[1], a[2], a[3], a[4], a[5], None, None, a[6], None, None, None, C.byref(c), 0, 0, None) == -1
    if not any(k.endswith(("row", "_batch")) for k in wrong):
        assert lib.rp_selective_scan_saved_elems(C.byref(c), 0) == -1 and lib.rp_selective_scan_ws_bytes(C.byref(c), 0, 1) == -1


def test_scan_refuses_bad_calls():
    lib, c = rpb.load(), scan()
    y, x, dt, A, B, Cm, z = (at(2048 * i) for i in range(7))

    def call(y=y, x=x, dt=dt, A=A, B=B, Cm=Cm, z=z, c=c, saved=None, h_out=None, dtype=0, device=0):
        return lib.rp_selective_scan_ex(y, h_out, saved, x, dt, A, B, Cm, None, None, z, None, None, None, C.byref(c) if c else None, dtype, device, None)

    for missing in ("y", "x", "dt", "A", "B", "Cm", "c"):
        assert call(**{missing: None}) == -1
    assert call(device=-1) == -1 and call(dtype=4) == -1
    for other in (x, dt, B, Cm, z):
        assert call(y=other) == -1                                  # y over an operand
    assert call(c=scan(batch=1, length=4096)) == -1                 # split, and no workspace
    assert call(saved=A, h_out=A) == -1

    def grad(dy=at(14000), saved=at(20000), ws=at(30000), z=z, dtype=0, device=0, c=c, dh_out=None, **out):
        names = ("dx", "ddt", "dA", "dB", "dC", "dD", "ddt_bias", "dz", "dh_in")
        return lib.rp_selective_scan_grad_ex(*(out.get(k) for k in names), 0, dy, dh_out, x, dt, A, B, Cm, None, None, z, None, saved, ws,
                                             C.byref(c), dtype, device, None)

    free = at(40000)
    assert grad() == -1                                             # nothing wanted
    assert grad(dx=free, dy=None) == -1 and grad(dx=free, saved=None) == -1 and grad(dx=free, ws=None) == -1
    assert grad(dz=free, z=None) == -1
    assert grad(dx=free, device=-1) == -1 and grad(dx=free, dtype=7) == -1
    assert grad(dx=x) == -1 and grad(ddt=at(14000)) == -1 and grad(dB=B) == -1          # over an operand, over dy
    assert grad(dx=free, ddt=free) == -1                            # over one another
    assert grad(dx=free, c=scan(dx_row=5)) == -1 and grad(dB=free, c=scan(db_batch=3)) == -1
    assert grad(dh_in=free, dh_out=free) == -1


def norm(rows=4, channels=8, eps=1e-5, **over):
    c = rpb.RpbBlockNorm()
    rpb.load().rpb_block_norm_packed(C.byref(c), rows, channels, eps)
    for k, v in over.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("wrong", [dict(rows=0), dict(channels=0), dict(channels=8193), dict(eps=-1.0), dict(eps=float("nan")), dict(out_row=7),
                                   dict(y_row=-8), dict(u_row=-1), dict(r_row=-1), dict(rows=1 << 31), dict(u_row=1 << 31)])
def test_norm_refuses_bad_geometry(wrong):
    lib, c = rpb.load(), norm(**wrong)
    a = [at(2048 * i) for i in range(6)]
    assert lib.rp_block_norm_ex(a[0], a[1], a[2], None, None, None, a[3], a[4], C.byref(c), 0, 0, None) == -1
    if not any(k.endswith("row") for k in wrong):
        assert lib.rp_block_norm_ws_bytes(C.byref(c), 0) == -1


def test_norm_refuses_bad_calls():
    lib, c = rpb.load(), norm()
    out, y, u, z, r, w = (at(2048 * i) for i in range(6))
    call = lambda out=out, y=y, u=u, wb=w, dtype=0, device=0, g=c: lib.rp_block_norm_ex(out, y, u, z, None, None, r, wb, C.byref(g) if g else None,   # noqa: E731
                                                                                      dtype, device, None)
    assert call(u=None) == -1 and call(out=None, y=None) == -1 and call(wb=None) == -1 and call(g=None) == -1
    assert call(device=-1) == -1 and call(dtype=-1) == -1
    assert call(out=u) == -1 and call(y=r) == -1 and call(out=y) == -1 and call(y=z) == -1
    names = ("du", "dz", "dr", "dw_after", "dscale", "dw_before")

    def grad(dout=at(13000), dy=at(14000), z=z, wa=w, sc=w, wb=w, ws=at(20000), **outs):
        return lib.rp_block_norm_grad_ex(*(outs.get(k) for k in names), 0, dout, dy, u, z, wa, sc, r, wb, ws, C.byref(c), 0, 0, None)

    free = at(30000)
    assert grad() == -1 and grad(du=free, dout=None, dy=None) == -1 and grad(du=free, wb=None) == -1
    assert grad(dz=free, z=None) == -1 and grad(dw_after=free, wa=None) == -1 and grad(dscale=free, sc=None) == -1
    assert grad(dw_before=free, dy=None) == -1 and grad(dw_before=free, ws=None) == -1
    assert grad(du=u) == -1 and grad(dr=at(13000)) == -1 and grad(du=free, dr=free) == -1


def tensor(shape, strides, dtype=rpb.F32, data=None):
    """A Tensor struct as RecPulse lays it out, on device 0, over memory that no test reaches."""
    t = rpb._lib.CTensor()
    t.dtype, t.ndim, t.device_id, t.refcount, t.size = dtype, len(shape), 0, 1, int(np.prod(shape))
    t.shape, t.strides = (C.c_int * len(shape))(*shape), (C.c_int * len(strides))(*strides)
    t.data = data if data is not None else BUF.ctypes.data
    return t


@pytest.mark.parametrize("shape,strides", [((4, 1, 5, 8), (80, 80, 8, 1)), ((4, 5, 1, 8), (80, 8, 8, 1)), ((4, 5, 8), (80, 8, 1)), ((3, 1, 4, 1, 8), (32, 0, 16, 8, 1)),
                                           ((4, 5, 8), (8, 0, 1)), ((2, 8), (8, 2)), ((2, 8), (-8, 1))])
def test_norm_nodes_refuse_rows_at_several_distances(shape, strides, capfd):
    lib = rpb.load()
    u, w = tensor(shape, strides), tensor((8,), (1,))
    good = tensor(shape, tuple(int(np.prod(shape[d + 1:])) for d in range(len(shape))))
    assert not lib.op_rms_norm(C.byref(u), C.byref(w), 1e-5)
    assert not lib.op_gated_norm(C.byref(u), None, C.byref(w), None, None, 1e-5)
    assert not lib.op_gated_norm(C.byref(good), None, C.byref(w), None, C.byref(u), 1e-5)
    assert capfd.readouterr().err.count("rows at one distance") == 3


def test_nodes_refuse_empty_dimensions(capfd):
    """A Tensor with no elements (RecPulse's own can be had) is refused, not divided by."""
    lib = rpb.load()
    x, empty = tensor((2, 5, 8), (40, 8, 1)), tensor((2, 5, 0), (0, 0, 1))
    A, w = tensor((8, 4), (4, 1)), tensor((8,), (1,))
    none = tensor((8, 0), (0, 1))
    by = C.byref
    assert not lib.op_selective_scan(by(x), by(x), by(none), by(x), by(x), None, None, None, 1)
    assert not lib.op_selective_scan(by(x), by(x), by(A), by(empty), by(empty), None, None, None, 1)
    assert not lib.op_selective_scan(by(empty), by(empty), by(none), by(x), by(x), None, None, None, 1)
    for t in (empty, tensor((0, 8), (8, 1)), tensor((0,), (1,))):
        assert not lib.op_rms_norm(by(t), by(w), 1e-5) and not lib.op_gated_norm(by(t), None, None, None, None, 1e-5)
    assert not lib.op_causal_conv(by(empty), by(tensor((0, 4), (4, 1))), None, 1)
    assert not lib.op_causal_conv(by(x), by(none), None, 1)
    assert "cudaMalloc" not in capfd.readouterr().err


def overlap_refused(capfd, call, *names):
    """The call is refused, for an overlap of the two named buffers (in any order)."""
    capfd.readouterr()
    assert call() == -1
    err = capfd.readouterr().err
    assert "overlaps" in err and all(f" {n} " in err.replace("\n", " ") for n in names), (names, err)


def test_convolution_refuses_outputs_over_packed_operands(capfd):
    lib, c = rpb.load(), conv()                                    # x, y 320 bytes, w 128, bias 32, states 192
    base = dict(y=at(0), so=None, x=at(8192), w=at(16384), b=at(17000), si=at(18000), n=at(19000))
    call = lambda **k: lambda: lib.rp_causal_conv_ex(*{**base, **k}.values(), C.byref(c), 0, 0, None)          # noqa: E731
    overlap_refused(capfd, call(y=at(16384 + 124)), "y", "w")
    overlap_refused(capfd, call(y=at(17000 - 316)), "y", "bias")
    overlap_refused(capfd, call(y=at(18000)), "y", "state_in")
    overlap_refused(capfd, call(y=at(19004)), "y", "lengths")
    overlap_refused(capfd, call(so=at(8192)), "state_out", "x")
    overlap_refused(capfd, call(so=at(316)), "state_out", "y")
    overlap_refused(capfd, call(so=at(18000 + 188)), "state_out", "state_in")      # in place it may be, shifted not
    overlap_refused(capfd, call(so=at(18000 - 4)), "state_out", "state_in")
    grads = dict(dx=at(0), dw=at(1000), db=at(2000), ds=at(3000), acc=0, dy=at(4000), dso=at(5000), x=at(8192), w=at(16384), b=at(17000), si=at(18000),
                 n=None, ws=at(30000))
    grad = lambda **k: lambda: lib.rp_causal_conv_grad_ex(*{**grads, **k}.values(), C.byref(c), 0, 0, None)    # noqa: E731
    overlap_refused(capfd, grad(dx=at(16384)), "dx", "w")
    overlap_refused(capfd, grad(dw=at(16384 + 4)), "dw", "w")
    overlap_refused(capfd, grad(dw=at(4000)), "dw", "dy")
    overlap_refused(capfd, grad(db=at(1124)), "dbias", "dw")
    overlap_refused(capfd, grad(ds=at(18000 + 4)), "dstate_in", "state_in")
    overlap_refused(capfd, grad(ds=at(5000)), "dstate_in", "dstate_out")
    overlap_refused(capfd, grad(ws=at(8192)), "ws", "x")
    overlap_refused(capfd, grad(ws=at(0)), "ws", "dx")


def test_scan_refuses_outputs_over_packed_operands(capfd):
    lib, c = rpb.load(), scan()                                    # rows 320 bytes each, A 128, D 32, states 256
    a = [at(2048 * i) for i in range(16)]
    base = dict(y=a[0], ho=None, saved=None, x=a[1], dt=a[2], A=a[3], B=a[4], C=a[5], D=a[6], bias=a[7], z=a[8], hi=a[9], n=a[10], ws=None)
    call = lambda **k: lambda: lib.rp_selective_scan_ex(*{**base, **k}.values(), C.byref(c), 0, 0, None)       # noqa: E731
    for name, i in (("A", 3), ("D", 6), ("dt_bias", 7), ("h_in", 9), ("lengths", 10)):
        overlap_refused(capfd, call(y=a[i]), "y", name)
    overlap_refused(capfd, call(ho=at(2048 * 9 + 4)), "h_out", "h_in")
    overlap_refused(capfd, call(ho=a[1]), "h_out", "x")
    overlap_refused(capfd, call(ho=at(316)), "h_out", "y")
    overlap_refused(capfd, call(saved=at(2048 * 9 + 252)), "saved", "h_in")
    overlap_refused(capfd, call(saved=a[11], ho=at(2048 * 11 + 4)), "saved", "h_out")
    long = scan(batch=1, length=300, channels=4, states=1, groups=1)
    split = lambda ws: lambda: lib.rp_selective_scan_ex(at(0), None, None, at(8192), at(16384), at(24000), at(26000), at(30000), None, None, None, None,     # noqa: E731
                                                        None, ws, C.byref(long), 0, 0, None)
    assert lib.rp_selective_scan_ws_bytes(C.byref(long), 0, 0) > 0
    overlap_refused(capfd, split(at(8192)), "ws", "x")
    names = ("dx", "ddt", "dA", "dB", "dC", "dD", "ddt_bias", "dz", "dh_in")
    outs = {k: at(32768 + 1024 * i) for i, k in enumerate(names)}
    rest = dict(acc=0, dy=a[0], dho=a[11], x=a[1], dt=a[2], A=a[3], B=a[4], C=a[5], D=a[6], bias=a[7], z=a[8], n=None, saved=a[12], ws=at(50000))
    grad = lambda **k: lambda: lib.rp_selective_scan_grad_ex(*{**outs, **rest, **k}.values(), C.byref(c), 0, 0, None)      # noqa: E731
    overlap_refused(capfd, grad(dA=a[3]), "dA", "A")
    overlap_refused(capfd, grad(dD=outs["dA"]), "dD", "dA")
    overlap_refused(capfd, grad(ddt_bias=a[1]), "ddt_bias", "x")
    overlap_refused(capfd, grad(dh_in=at(2048 * 11 + 4)), "dh_in", "dh_out")
    overlap_refused(capfd, grad(dx=a[12]), "dx", "saved")
    overlap_refused(capfd, grad(ws=a[0]), "ws", "dy")
    overlap_refused(capfd, grad(ws=outs["dx"]), "ws", "dx")


def test_norm_refuses_outputs_over_weights(capfd):
    lib, c = rpb.load(), norm()                                    # rows 128 bytes, weights 32
    base = dict(out=at(0), y=at(1000), u=at(2000), z=at(3000), wa=at(4000), sc=at(4100), r=at(5000), wb=at(4200))
    call = lambda **k: lambda: lib.rp_block_norm_ex(*{**base, **k}.values(), C.byref(c), 0, 0, None)           # noqa: E731
    overlap_refused(capfd, call(out=at(4000)), "out", "w_after")
    overlap_refused(capfd, call(y=at(4228)), "y", "w_before")
    overlap_refused(capfd, call(out=at(4100 - 124), wa=at(6000)), "out", "scale")
    overlap_refused(capfd, call(y=at(124)), "y", "out")
    outs = dict(du=at(10000), dz=at(11000), dr=at(12000), dwa=at(13000), dsc=at(13100), dwb=at(13200), acc=0, dout=at(14000), dy=at(15000))
    rest = {k: base[k] for k in ("u", "z", "wa", "sc", "r", "wb")}
    grad = lambda **k: lambda: lib.rp_block_norm_grad_ex(*{**outs, **rest, "ws": at(20000), **k}.values(), C.byref(c), 0, 0, None)     # noqa: E731
    overlap_refused(capfd, grad(dwa=at(4000)), "dw_after", "w_after")
    overlap_refused(capfd, grad(dsc=at(13000)), "dscale", "dw_after")
    overlap_refused(capfd, grad(du=at(4200)), "du", "w_before")
    overlap_refused(capfd, grad(dwb=at(2000)), "dw_before", "u")
    overlap_refused(capfd, grad(ws=at(3000)), "ws", "z")
    overlap_refused(capfd, grad(ws=at(13000)), "ws", "dw_after")


@pytest.mark.parametrize("dtype,size", [(rpb.F32, 4), (rpb.F64, 8), (rpb.F16, 2), (rpb.BF16, 2)])
def test_buffers_off_their_elements_are_refused(dtype, size, capfd):
    """The GPU faults on them, so no call with one may reach it."""
    lib = rpb.load()
    wide = 8 if dtype == rpb.F64 else 4                            # of sums, states and workspaces
    start = (-BUF.ctypes.data) % 16

    def refused(fn, names, sizes, tail):
        """Every buffer in turn one byte (half an element) off, the others where they belong."""
        places = [None if s is None else at(start + 2960 * i) for i, s in enumerate(sizes)]
        for i, (name, s) in enumerate(zip(names, sizes)):
            if s is None or name is None:
                continue
            for shift in {1, s // 2}:
                now = list(places)
                now[i] = at(start + 2960 * i + shift)
                capfd.readouterr()
                assert fn(*now, *tail) == -1
                assert f"{name} is not aligned" in capfd.readouterr().err, name

    c = conv()
    tail = (C.byref(c), dtype, 0, None)
    refused(lib.rp_causal_conv_ex, ("y", "state_out", "x", "w", "bias", "state_in", "lengths"), (size,) * 6 + (4,), tail)
    grad = lambda *p: lib.rp_causal_conv_grad_ex(*p[:4], 0, *p[4:])                                # noqa: E731
    refused(grad, ("dx", "dw", "dbias", "dstate_in", "dy", "dstate_out", "x", "w", "bias", "state_in", "lengths", "ws"), (size,) * 10 + (4, wide), tail)
    c2 = scan()
    tail = (C.byref(c2), dtype, 0, None)
    refused(lib.rp_selective_scan_ex, ("y", "h_out", "saved", "x", "dt", "A", "B", "C", "D", "dt_bias", "z", "h_in", "lengths", "ws"),
            (size, wide, wide, size, size, wide, size, size, wide, wide, size, wide, 4, None), tail)
    grad2 = lambda *p: lib.rp_selective_scan_grad_ex(*p[:9], 0, *p[9:])                            # noqa: E731
    refused(grad2, ("dx", "ddt", "dA", "dB", "dC", "dD", "ddt_bias", "dz", "dh_in", "dy", "dh_out", "x", "dt", "A", "B", "C", "D", "dt_bias", "z", "lengths"),
            (size, size, wide, size, size, wide, wide, size, wide, size, wide, size, size, wide, size, size, wide, wide, size, 4, wide, wide), tail)
    c3 = norm()
    tail = (C.byref(c3), dtype, 0, None)
    refused(lib.rp_block_norm_ex, ("out", "y", "u", "z", "w_after", "scale", "r", "w_before"), (size,) * 8, tail)
    grad3 = lambda *p: lib.rp_block_norm_grad_ex(*p[:6], 0, *p[6:])                                # noqa: E731
    refused(grad3, ("du", "dz", "dr", "dw_after", "dscale", "dw_before", "dout", "dy", "u", "z", "w_after", "scale", "r", "w_before", "ws"),
            (size,) * 14 + (wide,), tail)
