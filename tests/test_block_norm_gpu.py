"""rp_block_norm_ex / rp_block_norm_grad_ex against the formulas in float64: types, row lengths, every part left out in turn,
strided rows, accumulation, streams and graphs."""
import ctypes as C

import pytest
import torch

import recpulse_b200 as rpb
from seq_helpers import CODE, TYPES, close, ptr, same_bits, stream, unit

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.fixture(scope="module")
def lib():
    lib = rpb.load()
    yield lib
    assert lib.rpb_device_status(0) == 0


def make(rows, d, dtype, seed, without=()):
    gen = torch.Generator().manual_seed(seed)
    t = TYPES[dtype]
    rand = lambda *s: torch.randn(*s, generator=gen).to(t).cuda()           # noqa: E731
    u, z = rand(rows, 2 * d).split(d, dim=1)
    s = {"u": u, "z": z, "r": 2 * rand(rows, d), "w_after": 1 + 0.2 * rand(d), "w_before": 1 + 0.2 * rand(d), "scale": 0.5 * rand(d),
         "dout": rand(rows, d), "dy": rand(rows, d)}
    return {k: (None if k in without else v) for k, v in s.items()}


def reference(s, dtype):
    """Values and gradients in float64 with the slack of their arithmetic.  A sum over a row of d values is taken as d / (a
    warp's lanes ...) short sums and then as a tree: below `steps` roundings; a mean of squares halves into its root."""
    u = unit(dtype)
    f = {k: (v.double().cpu() if v is not None else None) for k, v in s.items()}
    x = f["u"]
    rows, d = x.shape
    eps = float(torch.tensor(EPS, dtype=torch.float32))
    steps = 24 + d / 256
    one = torch.ones(d, dtype=torch.float64)
    if f["z"] is not None:
        z = f["z"]
        sig = torch.sigmoid(z)
        # the exponential within 4 + |z| steps, a sum, a quotient; 0 below the normal range
        sig_err = sig * (1 - sig) * (4 + z.abs()) * 2 * u + 3 * u * sig + 2.0 ** -126
        gate, gate_err = z * sig, z.abs() * (sig_err + u * sig)
        slope, slope_err = sig * (1 + z * (1 - sig)), sig_err * (1 + z.abs()) + 6 * u * sig * (1 + z.abs() * (1 - sig))
    else:
        gate, gate_err = torch.ones_like(x), torch.zeros_like(x)
    v, v_err = x * gate, x.abs() * (gate_err + u * gate.abs())

    def inverse(a, a_err):
        """1 / root of the mean square, and its relative error"""
        mean = (a * a).mean(1, keepdim=True) + eps
        rel = ((2 * a.abs() * a_err).mean(1, keepdim=True) / mean + (steps + 3) * u) / 2 + 4 * u
        return mean.rsqrt(), rel

    wa, sc = f["w_after"] if f["w_after"] is not None else one, f["scale"] if f["scale"] is not None else one
    i1, rel1 = inverse(v, v_err) if f["w_after"] is not None else (torch.ones(rows, 1, dtype=torch.float64), torch.zeros(rows, 1, dtype=torch.float64))
    t, t_err = v * i1, v_err * i1 + (v * i1).abs() * (rel1 + u)
    add = sc * wa * t
    add_err = (sc * wa).abs() * t_err + 3 * u * add.abs()
    r = f["r"] if f["r"] is not None else torch.zeros_like(x)
    out, out_err = r + add, add_err + u * (r + add).abs()
    res = {"out": out, "out_slack": out_err}
    wb = f["w_before"]
    if wb is not None:
        i2, rel2 = inverse(out, out_err)
        q, q_err = out * i2, out_err * i2 + (out * i2).abs() * (rel2 + u)
        res["y"], res["y_slack"] = q * wb, q_err * wb.abs() + u * (q * wb).abs()
    rows_steps = 24 + rows / 4

    def back(m, m_err, q, q_err, i, rel):
        """i (m - q mean(m q)) and its error"""
        dot = (m * q).mean(1, keepdim=True)
        dot_err = (m_err * q.abs() + m.abs() * q_err + (steps + 3) * u * (m * q).abs()).mean(1, keepdim=True)
        inner = m - q * dot
        inner_err = m_err + q_err * dot.abs() + q.abs() * dot_err + 4 * u * ((q * dot).abs() + m.abs())
        return i * inner, i * inner_err + (i * (m.abs() + (q * dot).abs())) * (rel + 2 * u)

    total = f["dout"] if f["dout"] is not None else torch.zeros_like(x)
    total_err = torch.zeros_like(x)
    if f["dy"] is not None and wb is not None:
        dy = f["dy"]
        res["dw_before"] = (dy * q).sum(0)
        res["dw_before_slack"] = (dy.abs() * q_err + (rows_steps + 3) * u * (dy * q).abs()).sum(0)
        pull, pull_err = back(dy * wb, u * (dy * wb).abs(), q, q_err, i2, rel2)
        total, total_err = total + pull, pull_err + u * (total + pull).abs()
    res["dr"], res["dr_slack"] = total, total_err
    for name, m in (("dscale", wa), ("dw_after", sc)):
        res[name] = (total * m * t).sum(0)
        res[name + "_slack"] = (total_err * (m * t).abs() + (total * m).abs() * t_err + (rows_steps + 4) * u * (total * m * t).abs()).sum(0)
    m = total * sc * wa
    m_err = total_err * (sc * wa).abs() + 2 * u * m.abs()
    dv, dv_err = back(m, m_err, t, t_err, i1, rel1) if f["w_after"] is not None else (m, m_err)
    res["du"], res["du_slack"] = dv * gate, dv_err * gate.abs() + dv.abs() * (gate_err + 2 * u * gate.abs())
    if f["z"] is not None:
        res["dz"] = dv * x * slope
        res["dz_slack"] = dv_err * (x * slope).abs() + dv.abs() * x.abs() * (slope_err + 4 * u * slope.abs())
    return res


GRADS = ("du", "dz", "dr", "dw_after", "dscale", "dw_before")


def geometry(s, **over):
    rows, d = s["u"].shape
    c = rpb.RpbBlockNorm()
    rpb.load().rpb_block_norm_packed(C.byref(c), rows, d, EPS)
    for k in ("u", "z", "r"):
        if s[k] is not None:
            setattr(c, k + "_row", s[k].stride(0))
    for k, v in over.items():
        setattr(c, k, v)
    return c


def forward(lib, s, c, dtype):
    nan = lambda: torch.full(s["u"].shape, float("nan"), dtype=s["u"].dtype, device="cuda")       # noqa: E731
    out, y = nan(), nan() if s["w_before"] is not None else None
    assert lib.rp_block_norm_ex(ptr(out), ptr(y), ptr(s["u"]), ptr(s["z"]), ptr(s["w_after"]), ptr(s["scale"]), ptr(s["r"]), ptr(s["w_before"]),
                                C.byref(c), CODE[dtype], 0, stream()) == 0
    return {"out": out, "y": y}


def backward(lib, s, c, dtype, out=None, accumulate=0, ws=None):
    if out is None:
        nan = lambda like: torch.full(like.shape, float("nan"), dtype=like.dtype, device="cuda")      # noqa: E731
        have = {"du": s["u"], "dz": s["z"], "dr": s["u"], "dw_after": s["w_after"], "dscale": s["scale"],
                "dw_before": s["w_before"] if s["dy"] is not None else None}
        out = {k: nan(v) for k, v in have.items() if v is not None}
    if ws is None:
        ws = torch.full((lib.rp_block_norm_ws_bytes(C.byref(c), CODE[dtype]),), 255, dtype=torch.uint8, device="cuda")
    assert lib.rp_block_norm_grad_ex(*(ptr(out.get(k)) for k in GRADS), accumulate, ptr(s["dout"]), ptr(s["dy"]), ptr(s["u"]), ptr(s["z"]),
                                     ptr(s["w_after"]), ptr(s["scale"]), ptr(s["r"]), ptr(s["w_before"]), ptr(ws), C.byref(c), CODE[dtype], 0,
                                     stream()) == 0
    return out


def check(lib, s, dtype, what):
    ref, c = reference(s, dtype), geometry(s)
    for k, v in forward(lib, s, c, dtype).items():
        if v is not None:
            close(v, ref[k], ref[k + "_slack"], f"{what} {k}")
    got = backward(lib, s, c, dtype)
    for k, v in got.items():
        close(v, ref[k], ref[k + "_slack"], f"{what} {k}")
    again = backward(lib, s, c, dtype)
    assert all(same_bits(got[k], again[k]) for k in got), what


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 7), (2, 8), (5, 64), (33, 200), (2, 1000), (7, 1531), (3, 4096), (2, 8192), (9, 8191), (5, 4095), (700, 40), (40, 2999), (1300, 257)])
def test_forward_and_backward(lib, dtype, rows, d):
    check(lib, make(rows, d, dtype, rows * d), dtype, f"{dtype} {rows}x{d}")


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("without", [("z",), ("w_after",), ("scale",), ("r",), ("w_before", "dy"), ("dy",), ("dout",), ("z", "w_after", "scale", "r"),
                                     ("w_after", "scale", "z", "w_before", "dy")])
def test_parts_left_out(lib, dtype, without):
    check(lib, make(9, 72, dtype, 3, without), dtype, f"{dtype} without {without}")


def test_y_alone_is_a_plain_norm(lib):
    """out NULL: only the norm is written; also with unaligned rows."""
    s = make(6, 50, "float16", 4, ("z", "w_after", "scale", "r"))
    wide = torch.full((6, 53), float("nan"), dtype=torch.float16, device="cuda")
    c = geometry(s, y_row=53)
    assert lib.rp_block_norm_ex(None, C.c_void_p(wide.data_ptr() + 2), ptr(s["u"]), None, None, None, None, ptr(s["w_before"]), C.byref(c),
                                CODE["float16"], 0, stream()) == 0
    ref = reference(s, "float16")
    close(wide[:, 1:51], ref["y"], ref["y_slack"], "y")
    assert wide[:, 0].isnan().all() and wide[:, 51:].isnan().all()


@pytest.mark.parametrize("d", [40, 37])
@pytest.mark.parametrize("shift", [0, 3])
def test_one_row_for_all(lib, d, shift):
    """A row stride of 0 (one residual row under every row), at an offset from a boundary: nothing in front of it is read."""
    s = make(12, d, "bfloat16", 5)
    memory = torch.full((shift + d,), float("inf"), dtype=torch.bfloat16, device="cuda")
    memory[shift:] = s["r"][0]
    s["r"] = memory[shift:].expand(12, d)
    s["u"], s["z"] = s["u"].contiguous(), s["z"].contiguous()
    check(lib, s, "bfloat16", f"one row {d} {shift}")
    first = torch.full((shift + 12 * d,), float("nan"), dtype=torch.bfloat16, device="cuda")
    first[shift:] = s["u"].reshape(-1)
    s = make(12, d, "bfloat16", 5, ("z", "r"))
    s["u"] = first[shift:].view(12, d)
    check(lib, s, "bfloat16", f"offset rows {d} {shift}")


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_accumulates_and_leaves_out(lib, dtype):
    s = make(19, 136, dtype, 6)
    ref, c = reference(s, dtype), geometry(s)
    first = {k: torch.randn(ref[k].shape, generator=torch.Generator().manual_seed(2)).to(s["u"].dtype).cuda() for k in GRADS}
    have = {k: v.clone() for k, v in first.items()}
    backward(lib, s, c, dtype, have, 63)
    fresh = backward(lib, s, c, dtype)
    for k in GRADS:
        want = ref[k] + first[k].double().cpu()
        close(have[k], want, ref[k + "_slack"] + unit(dtype) * want.abs(), k)
        alone = {k: torch.zeros_like(fresh[k])}
        backward(lib, s, c, dtype, alone)
        assert same_bits(alone[k], fresh[k]), k


def test_gradients_against_differences(lib):
    dtype = "float64"
    s = {k: v.contiguous() for k, v in make(3, 6, dtype, 8).items()}
    c = geometry(s)
    got = backward(lib, s, c, dtype)

    def total():
        f = forward(lib, s, c, dtype)
        return float((f["out"] * s["dout"]).sum() + (f["y"] * s["dy"]).sum())

    step = 1e-5
    for name, key in (("u", "du"), ("z", "dz"), ("r", "dr"), ("w_after", "dw_after"), ("scale", "dscale"), ("w_before", "dw_before")):
        flat, g = s[name].view(-1), got[key].reshape(-1)
        for i in range(flat.numel()):
            keep = float(flat[i])
            flat[i] = keep + step; hi = total()
            flat[i] = keep - step; lo = total()
            flat[i] = keep
            # step^2 times third derivatives of order 10 (rows of 6), and the rounding of sums below 1e2 over 2 step
            assert abs((hi - lo) / (2 * step) - float(g[i])) < 5e-8, (name, i)


def test_replayed_from_a_graph_on_another_stream(lib):
    dtype = "bfloat16"
    s = {k: v.contiguous() for k, v in make(70, 264, dtype, 9).items()}
    c = geometry(s)
    ws = torch.empty(lib.rp_block_norm_ws_bytes(C.byref(c), CODE[dtype]), dtype=torch.uint8, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        got = {**forward(lib, s, c, dtype), **backward(lib, s, c, dtype, ws=ws)}
    for seed in range(2):
        s["u"].copy_(torch.randn(s["u"].shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        ref = reference(s, dtype)
        for k, v in got.items():
            close(v, ref[k], ref[k + "_slack"], k)


@pytest.mark.parametrize("dtype,rows,d", [("float32", 5, 4093), ("float32", 5, 8191), ("float64", 5, 2047), ("float64", 3, 8189), ("float16", 9, 8191),
                                          ("bfloat16", 9, 8187), ("float32", 3, 8192), ("float64", 2, 8192), ("bfloat16", 3, 8192)])
@pytest.mark.parametrize("shift", [0, 1])
def test_wide_rows_and_their_weights(lib, dtype, rows, d, shift):
    """Packed operands with rows too wide for shared memory: rows that begin off a 16-byte boundary meet weights that lie on one,
    and (shift) weights that begin off one meet rows that do not."""
    s = {k: v.contiguous() for k, v in make(rows, d, dtype, rows + d).items()}
    for k in ("w_after", "scale", "w_before"):
        memory = torch.full((shift + d,), float("nan"), dtype=s[k].dtype, device="cuda")
        memory[shift:] = s[k]
        s[k] = memory[shift:]
    check(lib, s, dtype, f"{dtype} {rows}x{d} weights {shift} off")
