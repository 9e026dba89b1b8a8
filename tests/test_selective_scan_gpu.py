"""rp_selective_scan_ex / rp_selective_scan_grad_ex against the recurrence in float64: types, state counts, groups, lengths,
strided column blocks, split sequences, single tokens, accumulation, streams and graphs."""
import ctypes as C

import pytest
import torch

import recpulse_b200 as rpb
from seq_helpers import CODE, TYPES, acc_type, close, overflowed, ptr, same_bits, stream, unit

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    lib = rpb.load()
    yield lib
    assert lib.rpb_device_status(0) == 0


def make(batch, length, d, n, groups, dtype, seed, state=False, gate=True, skip=True, bias=True):
    gen = torch.Generator().manual_seed(seed)
    t, a = TYPES[dtype], acc_type(dtype)
    rand = lambda *s: torch.randn(*s, generator=gen)                        # noqa: E731
    s = {}
    x, z = rand(batch, length, 2 * d).to(t).cuda().split(d, dim=2)
    s["x"], s["z"] = x, z if gate else None
    s["dt"] = (0.7 * rand(batch, length, d) - 1).to(t).cuda()
    _, s["B"], s["C"] = rand(batch, length, 3 + 2 * groups * n).to(t).cuda().split([3, groups * n, groups * n], dim=2)
    s["A"] = (-torch.arange(1, n + 1) * torch.exp(0.2 * rand(d, n)) * 0.5).to(a).cuda()
    s["D"] = rand(d).to(a).cuda() if skip else None
    s["dt_bias"] = (0.5 * rand(d)).to(a).cuda() if bias else None
    s["h"] = rand(batch, d, n).to(a).cuda() if state else None
    s["dy"] = rand(batch, length, d).to(t).cuda()
    s["dh"] = rand(batch, d, n).to(a).cuda() if state else None
    return s


def reference(s, n, groups, softplus, lengths=None, grad=False, dtype="float32"):
    """The recurrence row by row in float64; next to every value the slack that its arithmetic in float32 (float64) may
    cost, from the same recurrence on absolute values: a product of decays carries the relative error of its exponent
    (|delta A| twice rounded, an exponential within 4 steps), every other step one rounding.  An exponential below the
    normal range is stored as 0, so each also carries an absolute error of the smallest normal number, `tiny`."""
    u, tiny = unit(dtype), torch.finfo(acc_type(dtype)).tiny
    f = {k: (v.double().cpu() if v is not None else None) for k, v in s.items()}
    x, A = f["x"], f["A"]
    batch, length, d = x.shape
    zero = torch.zeros(d, dtype=torch.float64)
    D, bias = f["D"] if f["D"] is not None else zero, f["dt_bias"] if f["dt_bias"] is not None else zero
    raw = f["dt"] + bias
    delta = raw.clamp(min=0) + torch.log1p(torch.exp(-raw.abs())) if softplus else raw
    # raw: one rounding; softplus has slope sigmoid <= 1 and its own few steps
    delta_err = u * (raw.abs() * torch.sigmoid(raw) * (1 if softplus else 0) + (raw.abs() if not softplus else 0) + 12 * delta.abs()) + tiny
    ends = torch.tensor([min(max(int(v), 0), length) for v in lengths]) if lengths is not None else torch.full((batch,), length)
    live = torch.arange(length)[None, :, None] < ends[:, None, None]
    delta, delta_err, x = delta * live, delta_err * live, torch.where(live, x, 0.0)
    spread = lambda v, t: torch.where(live[:, t], v[:, t], 0.0).reshape(batch, groups, n).repeat_interleave(d // groups, dim=1)     # noqa: E731
    h = f["h"] if f["h"] is not None else torch.zeros(batch, d, n, dtype=torch.float64)
    e = torch.zeros_like(h)                      # error of h
    hs, es, core, core_err = [h], [e], torch.zeros_like(x), torch.zeros_like(x)
    decays = []
    for t in range(length):
        step, serr = delta[:, t, :, None], delta_err[:, t, :, None]
        a = torch.exp(step * A)
        aerr = a * ((serr + 3 * u * step.abs()) * A.abs() + 4 * u) + tiny
        Bt, Ct = spread(f["B"], t), spread(f["C"], t)
        feed = step * x[:, t, :, None] * Bt
        ferr = (serr * x[:, t, :, None] * Bt).abs() + 2 * u * feed.abs()
        e = torch.where(live[:, t, :, None], a * e + aerr * h.abs() + ferr + 2 * u * ((a * h).abs() + feed.abs()), e)
        h = torch.where(live[:, t, :, None], a * h + feed, h)
        e = overflowed(e, dtype, h, a, feed)
        hs.append(h); es.append(e); decays.append((a, aerr))
        core[:, t] = (h * Ct).sum(-1) + D * x[:, t]
        core_err[:, t] = (e * Ct.abs()).sum(-1) + (n + 3) * u * ((h * Ct).abs().sum(-1) + (D * x[:, t]).abs())
        core_err[:, t] = overflowed(core_err[:, t], dtype, (h * Ct).abs().sum(-1))
    out = {"h": h, "h_slack": e}
    if f["z"] is not None:
        z = torch.where(live, f["z"], 0.0)
        sig = torch.sigmoid(z)
        sig_err = sig * (1 - sig) * (4 + z.abs()) * 2 * u + 3 * u * sig + tiny
        gate, gate_err = z * sig, z.abs() * (sig_err + u * sig)
        slope = sig * (1 + z * (1 - sig))
        slope_err = sig_err * (1 + z.abs()) + 6 * u * (sig + (z * sig * (1 - sig)).abs())
    else:
        gate, gate_err = torch.ones_like(x), torch.zeros_like(x)
    out["y"] = torch.where(live, core * gate, 0.0)
    out["y_slack"] = core_err * gate.abs() + core.abs() * (gate_err + u * gate.abs())
    if not grad:
        return out
    dy = torch.where(live, f["dy"], 0.0)
    if f["z"] is not None:
        out["dz"] = dy * core * slope
        out["dz_slack"] = dy.abs() * (core_err * slope.abs() + core.abs() * (slope_err + 3 * u * slope.abs()))
        out["dz_slack"] = overflowed(out["dz_slack"], dtype, dy * core)
    dy, dy_err = dy * gate, dy.abs() * (gate_err + u * gate.abs())
    for k in ("dx", "ddt"):
        out[k], out[k + "_slack"] = torch.zeros_like(x), torch.zeros_like(x)
    for k in ("dB", "dC"):
        out[k], out[k + "_slack"] = (torch.zeros(batch, length, groups * n, dtype=torch.float64) for _ in range(2))
    out["dA"], out["dA_slack"] = torch.zeros_like(A), torch.zeros_like(A)
    by_group = lambda v: v.reshape(batch, groups, d // groups, n).sum(2).reshape(batch, -1)       # noqa: E731
    g = f["dh"] if f["dh"] is not None else torch.zeros_like(h)
    g = g.clone()
    ge = torch.zeros_like(g)
    total_dA = torch.zeros_like(A)
    sums = 64 + d // groups + batch * length        # no sum here has more steps than this
    for t in range(length - 1, -1, -1):
        on = live[:, t, :, None]
        a, aerr = decays[t]
        step, serr = delta[:, t, :, None], delta_err[:, t, :, None]
        Bt, Ct, xt = spread(f["B"], t), spread(f["C"], t), x[:, t, :, None]
        gy, gye = dy[:, t, :, None], dy_err[:, t, :, None]
        dh = g + gy * Ct
        dhe = ge + (gye * Ct).abs() + 2 * u * (g.abs() + (gy * Ct).abs())
        dhe = overflowed(dhe, dtype, dh, dh * a)
        out["dC"][:, t] = by_group(gy * hs[t + 1])
        out["dC_slack"][:, t] = by_group(gye * hs[t + 1].abs() + gy.abs() * es[t + 1] + sums * u * (gy * hs[t + 1]).abs())
        out["dB"][:, t] = by_group(dh * step * xt)
        out["dB_slack"][:, t] = by_group((dhe * step * xt).abs() + (dh * serr * xt).abs() + sums * u * (dh * step * xt).abs())
        inner = (dh * Bt).sum(-1)
        inner_err = (dhe * Bt.abs()).sum(-1) + (n + 2) * u * (dh * Bt).abs().sum(-1)
        da = dh * a * hs[t]
        dae = dhe * (a * hs[t]).abs() + dh.abs() * (aerr * hs[t].abs() + a * es[t]) + 3 * u * da.abs()
        dae = overflowed(dae, dtype, da, da * A, da * step)
        inner_err = overflowed(inner_err, dtype, (dh * Bt).abs().sum(-1))
        dd = (da * A).sum(-1) + inner * x[:, t]
        dd_err = (dae * A.abs()).sum(-1) + (n + 2) * u * (da * A).abs().sum(-1) + inner_err * x[:, t].abs() + 3 * u * (inner * x[:, t]).abs()
        dd_err = overflowed(dd_err, dtype, dd, inner * x[:, t], (da * A).abs().sum(-1))
        if softplus:
            sg = torch.sigmoid(raw[:, t])
            dd_err = dd_err * sg + dd.abs() * (sg * (1 - sg) * (4 + 3 * raw[:, t].abs()) * 2 * u + 4 * u * sg + tiny)
            dd = dd * sg
        out["ddt"][:, t], out["ddt_slack"][:, t] = dd, dd_err
        out["dx"][:, t] = delta[:, t] * inner + D * dy[:, t]
        out["dx_slack"][:, t] = delta[:, t].abs() * inner_err + (delta_err[:, t] * inner).abs() + D.abs() * dy_err[:, t] + \
            3 * u * ((delta[:, t] * inner).abs() + (D * dy[:, t]).abs())
        out["dA"] += torch.where(on, da * step, 0.0).sum(0)
        out["dA_slack"] += (dae * step.abs() + da.abs() * serr + sums * u * (da * step).abs()).sum(0)
        for k, parts in (("dC", gy * hs[t + 1]), ("dB", dh * step * xt)):
            out[k + "_slack"][:, t] = overflowed(out[k + "_slack"][:, t], dtype, by_group(parts.abs()))
        total_dA = total_dA + torch.where(on, (da * step).abs(), 0.0).sum(0)
        g, ge = torch.where(on, dh * a, g), torch.where(on, dhe * a + dh.abs() * aerr + u * (dh * a).abs(), ge)
    out["dA_slack"] = overflowed(out["dA_slack"], dtype, total_dA)
    mask = live.double()
    out["ddt"], out["dx"] = out["ddt"] * mask, out["dx"] * mask
    out["dD"] = (dy * x).sum((0, 1))
    out["dD_slack"] = (dy_err * x.abs() + sums * u * (dy * x).abs()).sum((0, 1))
    out["ddt_bias"] = out["ddt"].sum((0, 1))
    out["ddt_bias_slack"] = (out["ddt_slack"] * mask + sums * u * out["ddt"].abs()).sum((0, 1))
    out["dh_in"], out["dh_in_slack"] = g, ge
    return out


def geometry(s, n, groups, softplus, **over):
    batch, length, d = s["x"].shape
    c = rpb.RpbScan()
    rpb.load().rpb_scan_packed(C.byref(c), batch, length, d, n, groups, softplus)
    for k, v in (("x", s["x"]), ("dt", s["dt"]), ("b", s["B"]), ("c", s["C"]), ("z", s["z"])):
        if v is not None:
            setattr(c, k + "_batch", v.stride(0)); setattr(c, k + "_row", v.stride(1))
    for k, v in over.items():
        setattr(c, k, v)
    return c


def nan(*shape, dtype):
    return torch.full(shape, float("nan"), dtype=dtype, device="cuda")


def forward(lib, s, c, dtype, lengths=None, keep=False, h_out=None):
    a = acc_type(dtype)
    y = nan(c.batch, c.len, c.channels, dtype=s["x"].dtype)
    h = nan(c.batch, c.channels, c.states, dtype=a) if h_out is None else h_out
    saved = nan(lib.rp_selective_scan_saved_elems(C.byref(c), CODE[dtype]), dtype=a) if keep else None
    size = lib.rp_selective_scan_ws_bytes(C.byref(c), CODE[dtype], 0)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda") if size else None
    assert lib.rp_selective_scan_ex(ptr(y), ptr(h), ptr(saved), ptr(s["x"]), ptr(s["dt"]), ptr(s["A"]), ptr(s["B"]), ptr(s["C"]), ptr(s["D"]),
                                    ptr(s["dt_bias"]), ptr(s["z"]), ptr(s["h"]), ptr(lengths), ptr(ws), C.byref(c), CODE[dtype], 0, stream()) == 0
    return y, h, saved


GRADS = ("dx", "ddt", "dA", "dB", "dC", "dD", "ddt_bias", "dz", "dh_in")


def backward(lib, s, c, dtype, saved, lengths=None, out=None, accumulate=0, ws=None):
    a, t = acc_type(dtype), s["x"].dtype
    if out is None:
        gn = c.groups * c.states
        out = {"dx": nan(c.batch, c.len, c.channels, dtype=t), "ddt": nan(c.batch, c.len, c.channels, dtype=t), "dA": nan(c.channels, c.states, dtype=a),
               "dB": nan(c.batch, c.len, gn, dtype=t), "dC": nan(c.batch, c.len, gn, dtype=t), "dD": nan(c.channels, dtype=a),
               "ddt_bias": nan(c.channels, dtype=a), "dz": nan(c.batch, c.len, c.channels, dtype=t) if s["z"] is not None else None,
               "dh_in": nan(c.batch, c.channels, c.states, dtype=a)}
    if ws is None:
        ws = torch.full((lib.rp_selective_scan_ws_bytes(C.byref(c), CODE[dtype], 1),), 255, dtype=torch.uint8, device="cuda")
    assert lib.rp_selective_scan_grad_ex(*(ptr(out.get(k)) for k in GRADS), accumulate, ptr(s["dy"]), ptr(s["dh"]), ptr(s["x"]), ptr(s["dt"]),
                                         ptr(s["A"]), ptr(s["B"]), ptr(s["C"]), ptr(s["D"]), ptr(s["dt_bias"]), ptr(s["z"]), ptr(lengths),
                                         ptr(saved), ptr(ws), C.byref(c), CODE[dtype], 0, stream()) == 0
    return out


def check(lib, s, n, groups, softplus, dtype, what, lengths=None, clean=None):
    """One forward and backward call against the recurrence; `clean`: the operands without what lies behind the lengths."""
    given = torch.tensor(lengths, dtype=torch.int32, device="cuda") if lengths is not None else None
    ref = reference(clean or s, n, groups, softplus, lengths, True, dtype)
    c = geometry(s, n, groups, softplus)
    y, h, saved = forward(lib, s, c, dtype, given, keep=True)
    close(y, ref["y"], ref["y_slack"], what + " y")
    close(h, ref["h"], ref["h_slack"], what + " h")
    y2, h2, _ = forward(lib, s, c, dtype, given)
    close(y2, ref["y"], ref["y_slack"], what + " y, nothing saved")
    close(h2, ref["h"], ref["h_slack"], what + " h, nothing saved")
    got = backward(lib, s, c, dtype, saved, given)
    for k in GRADS:
        if got[k] is not None:
            close(got[k], ref[k], ref[k + "_slack"], f"{what} {k}")
    again = backward(lib, s, c, dtype, saved, given)
    assert all(same_bits(got[k], again[k]) for k in GRADS if got[k] is not None), what + ": equal inputs, other bits"
    return c


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [1, 2, 4, 5, 8, 10, 16, 17, 24, 32, 33, 64])
def test_forward_and_backward(lib, dtype, n):
    for k, (batch, length, d, groups) in enumerate([(1, 1, 1, 1), (2, 3, 40, 1), (1, 33, 36, 3), (2, 70, 129, 1), (3, 17, 64, 2)]):
        s = make(batch, length, d, n, groups, dtype, 31 * n + k, state=k % 2 == 1, gate=k % 3 != 2, skip=k != 2, bias=k != 1)
        check(lib, s, n, groups, int(k != 4), dtype, f"{dtype} n={n} {batch}x{length}x{d}/{groups}")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,groups", [(4, 256, 1), (4, 144, 2), (8, 160, 1), (12, 64, 1), (16, 96, 1), (24, 80, 2), (24, 650, 2), (28, 16, 1), (32, 48, 1),
                                        (44, 40, 1), (60, 24, 1), (64, 16, 1)])
def test_aligned_layouts(lib, dtype, n, d, groups):
    """Every operand aligned for whole packs, states in whole groups of four but not in powers of two; the columns behind B and
    C hold infinities, which nothing may reach; several tiles, the last one ragged."""
    length = 75
    s = make(2, length, d, n, groups, dtype, n + d, state=True)
    for k in ("B", "C"):
        wide = torch.full((2, length, groups * n + 16), float("inf"), dtype=s[k].dtype, device="cuda")
        wide[:, :, :groups * n] = s[k]
        s[k] = wide[:, :, :groups * n]
    check(lib, s, n, groups, 1, dtype, f"{dtype} n={n} d={d}/{groups}")


@pytest.mark.parametrize("dtype,n", [("bfloat16", 16), ("float32", 16), ("float32", 3), ("float64", 10), ("float16", 40)])
def test_split_sequences(lib, dtype, n):
    """One sequence of few channels is split into chunks; same checks, with states entering and gradients leaving."""
    d, length = 24, 600
    s = make(1, length, d, n, 1, dtype, 7, state=True)
    c = check(lib, s, n, 1, 1, dtype, "split")
    assert lib.rp_selective_scan_ws_bytes(C.byref(c), CODE[dtype], 0) > 0          # it is split
    h = s["h"].clone()                                                              # the state in place
    _, want, _ = forward(lib, s, c, dtype)
    s["h"] = h
    forward(lib, s, c, dtype, h_out=h)
    assert torch.equal(h, want)


@pytest.mark.parametrize("dtype,length,ends", [("bfloat16", 50, [0, 1, 7, 8, 9, 49, 50]), ("float32", 300, [0, 1, 64, 65, 200, 299, 300]),
                                               ("float32", 1, [0, 1, 0, 1, 1, 0, 1])])
def test_lengths_of_a_padded_batch(lib, dtype, length, ends):
    """NaN and infinities behind a sequence reach nothing; the state is the one at its end."""
    batch, d, n = 7, 16, 8
    s = make(batch, length, d, n, 1, dtype, 3, state=True)
    dirty = {k: (v.clone() if v is not None else None) for k, v in s.items()}
    for b, end in enumerate(ends):
        for k, bad in (("x", "nan"), ("dt", "nan"), ("B", "inf"), ("C", "-inf"), ("z", "nan"), ("dy", "inf")):
            dirty[k][b, end:] = float(bad)
    given = [v if v else -3 for v in ends]
    given[-1] = 10 ** 6
    check(lib, dirty, n, 1, 1, dtype, "lengths", given, clean=s)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32", "float64"])
@pytest.mark.parametrize("batch,d,n,groups", [(1, 5, 1, 1), (3, 33, 16, 3), (8, 64, 10, 2), (5, 20, 64, 1)])
def test_tokens_continue_a_prompt(lib, dtype, batch, d, n, groups):
    """A prompt, then single tokens with the state in place, against the recurrence over the whole sequence."""
    length, prompt = 14, 9
    s = make(batch, length, d, n, groups, dtype, 77, gate=d != 33)
    ref = reference(s, n, groups, 1, dtype=dtype)
    part = lambda lo, hi, h: {k: (v[:, lo:hi] if v is not None and v.ndim == 3 and k not in ("h", "dh") else v) for k, v in {**s, "h": h}.items()}      # noqa: E731
    y, h, _ = forward(lib, part(0, prompt, None), geometry(part(0, prompt, None), n, groups, 1), dtype)
    got = [y]
    for t in range(prompt, length):
        now = part(t, t + 1, h)
        got.append(forward(lib, now, geometry(now, n, groups, 1), dtype, h_out=h)[0])
    close(torch.cat(got, dim=1), ref["y"], ref["y_slack"], "y")
    close(h, ref["h"], ref["h_slack"], "h")


def test_decays_at_the_edges(lib):
    """delta of 0 and of thousands, A of 0, far below and above 0: no overflow where the formula has none."""
    dtype, n, d = "float32", 4, 8
    s = make(1, 12, d, n, 1, dtype, 19, gate=False, bias=False)
    s["dt"][:] = torch.tensor([-200.0, -30.0, 0.0, 1e-3, 5.0, 80.0, 3000.0, -1.0, 20.0, 0.5, -90.0, 1.0])[None, :, None]
    s["A"][:] = torch.tensor([0.0, -1e-6, -50.0, -1e4])
    check(lib, s, n, 1, 1, dtype, "edges")
    s["dt"].clamp_(max=3)
    s["A"][:] = torch.tensor([0.3, 0.0, -1.0, 0.1])
    check(lib, s, n, 1, 1, dtype, "growing states")


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_accumulates_and_leaves_out(lib, dtype):
    batch, length, d, n, groups = 2, 21, 24, 6, 2
    s = make(batch, length, d, n, groups, dtype, 23, state=True)
    ref = reference(s, n, groups, 1, None, True, dtype)
    wide = d + 4
    c = geometry(s, n, groups, 1, dx_batch=length * wide, dx_row=wide)
    _, _, saved = forward(lib, s, c, dtype, keep=True)
    fresh = backward(lib, s, c, dtype, saved, out={"dx": torch.zeros(batch, length, wide, dtype=s["x"].dtype, device="cuda")[:, :, :d]})
    close(fresh["dx"], ref["dx"], ref["dx_slack"], "dx alone")
    gen = torch.Generator().manual_seed(1)
    first = {k: torch.randn(ref[k].shape, generator=gen).to(s["x"].dtype if k in ("dx", "ddt", "dB", "dC", "dz") else torch.float32).cuda()
             for k in GRADS if k != "dh_in"}
    have = {k: v.clone() for k, v in first.items()}
    c = geometry(s, n, groups, 1)
    backward(lib, s, c, dtype, saved, out=have, accumulate=255)
    for k in have:
        want = ref[k] + first[k].double().cpu()
        close(have[k], want, ref[k + "_slack"] + unit(dtype) * want.abs(), k)
    for k in GRADS:
        one = backward(lib, s, c, dtype, saved)
        alone = {k: torch.full_like(one[k], 3.0)}
        backward(lib, s, c, dtype, saved, out=alone)
        assert torch.equal(alone[k], one[k]), k


def test_gradients_against_differences(lib):
    dtype, n, d, groups, length = "float64", 3, 4, 2, 11
    s = make(2, length, d, n, groups, dtype, 29, state=True)
    s = {k: v.contiguous() for k, v in s.items()}
    c = geometry(s, n, groups, 1)
    _, _, saved = forward(lib, s, c, dtype, keep=True)
    got = backward(lib, s, c, dtype, saved)

    def total():
        y, h, _ = forward(lib, s, c, dtype)
        return float((y * s["dy"]).sum() + (h * s["dh"]).sum())

    step = 1e-5
    for name, key in (("x", "dx"), ("dt", "ddt"), ("A", "dA"), ("B", "dB"), ("C", "dC"), ("D", "dD"), ("dt_bias", "ddt_bias"), ("z", "dz"), ("h", "dh_in")):
        flat, g = s[name].view(-1), got[key].reshape(-1)
        for i in range(0, flat.numel(), 5):
            keep = float(flat[i])
            flat[i] = keep + step; hi = total()
            flat[i] = keep - step; lo = total()
            flat[i] = keep
            # step^2 times third derivatives of order 1, and the rounding of sums below 1e2 over 2 step
            assert abs((hi - lo) / (2 * step) - float(g[i])) < 5e-8, (name, i)


def test_replayed_from_a_graph_on_another_stream(lib):
    dtype, n, groups, length, d = "bfloat16", 16, 1, 200, 48
    s = make(1, length, d, n, groups, dtype, 37)
    s = {k: (v.contiguous() if v is not None else None) for k, v in s.items()}
    c = geometry(s, n, groups, 1)
    ws = torch.empty(lib.rp_selective_scan_ws_bytes(C.byref(c), CODE[dtype], 1), dtype=torch.uint8, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        y, h, saved = forward(lib, s, c, dtype, keep=True)
        got = backward(lib, s, c, dtype, saved, ws=ws)
    for seed in range(2):
        s["x"].copy_(torch.randn(s["x"].shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        ref = reference(s, n, groups, 1, None, True, dtype)
        close(y, ref["y"], ref["y_slack"], "y"); close(h, ref["h"], ref["h_slack"], "h")
        for k in GRADS:
            close(got[k], ref[k], ref[k + "_slack"], k)


@pytest.mark.parametrize("dtype,n,groups", [("float32", 4, 1), ("bfloat16", 16, 2), ("float64", 3, 1), ("float16", 33, 1)])
def test_zero_states_cross_fast_growing_chunks(lib, dtype, n, groups):
    """A split sequence part of which would let states grow beyond the type's range within a chunk: in front of the first x, and (for
    the gradients) behind the last dy.  The states there are 0 and stay it, so nothing overflows in the recurrence."""
    d, length = 12, 500
    s = make(1, length, d, n, groups, dtype, 45, gate=False, bias=False)
    s["A"][:] = 4.0 if dtype != "float64" else 32.0                 # a chunk is at least 64 rows: e^(64 * 0.5 * 4)
    s["dt"][:] = 0.5
    s["dt"][:, 400:] = 0.0003
    s["x"][:, :400] = 0
    c = geometry(s, n, groups, 0)
    assert lib.rp_selective_scan_ws_bytes(C.byref(c), CODE[dtype], 0) > 0          # it is split
    ref = reference(s, n, groups, 0, dtype=dtype)
    assert all(torch.isfinite(ref[k]).all() for k in ("y", "y_slack", "h", "h_slack"))
    y, h, _ = forward(lib, s, c, dtype)
    close(y, ref["y"], ref["y_slack"], "y")
    close(h, ref["h"], ref["h_slack"], "h")
    s["dt"] = s["dt"].flip(1).contiguous()
    s["x"][:] = 0
    s["dy"][:, 100:] = 0
    ref = reference(s, n, groups, 0, None, True, dtype)
    assert all(torch.isfinite(ref[k]).all() for k in ref)
    check(lib, s, n, groups, 0, dtype, "growing behind the gradients")


@pytest.mark.parametrize("dtype,length,ends", [("float32", 37, [37, 5, 0]), ("bfloat16", 70, [70, 33, 1]), ("float64", 21, [21, 8, 3]), ("float16", 9, [9, 9, 9]),
                                               ("float32", 300, [300, 100, 290])])
@pytest.mark.parametrize("infinite", [False, True])
def test_states_that_forget_at_once(lib, dtype, length, ends, infinite):
    """A at the end of its type's range, or infinite: every row's state is its own feed, also behind rows of a tile that are not part
    of the sequence, whose delta is 0."""
    d, n, a = 12, 6, acc_type(dtype)
    s = make(3, length, d, n, 1, dtype, 47, state=True)
    s["A"][:, ::2] = -1e30                                         # the same decays: 0 for every delta of a row
    ref = reference(s, n, 1, 1, ends, True, dtype)
    s["A"][:, ::2] = -float("inf") if infinite else -torch.finfo(a).max
    c, given = geometry(s, n, 1, 1), torch.tensor(ends, dtype=torch.int32, device="cuda")
    y, h, saved = forward(lib, s, c, dtype, given, keep=True)
    close(y, ref["y"], ref["y_slack"], "y")
    close(h, ref["h"], ref["h_slack"], "h")
    got = backward(lib, s, c, dtype, saved, given)
    for k in GRADS:
        if not (infinite and k in ("ddt", "ddt_bias")):             # 0 times A is part of these
            close(got[k], ref[k], ref[k + "_slack"], k)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d", [(4, 8), (16, 3)])
def test_an_infinite_gradient_of_A_stays_one(lib, dtype, n, d):
    """One infinite dy in the last tile of several: what the tiles in front of it add leaves dA the infinity that it is."""
    s = make(1, 100, d, n, 1, dtype, 53, state=True, gate=False)
    for k in ("B", "C", "h", "x", "D", "dy", "dh"):
        s[k] = s[k].abs() + 0.01
    s["A"][:] = -0.1
    s["dy"][:, 95] = float("inf")
    c = geometry(s, n, 1, 1)
    _, _, saved = forward(lib, s, c, dtype, keep=True)
    got = backward(lib, s, c, dtype, saved)
    assert (got["dA"] == float("inf")).all() and (got["dh_in"] == float("inf")).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [1, 2, 3, 5, 6, 9, 17, 20, 33, 62])
@pytest.mark.parametrize("length,d", [(1, 10), (45, 24), (400, 6)])
def test_one_infinite_row_of_each_channel(lib, dtype, n, length, d):
    """Channel c has one infinite x (then one infinite dy), with states, B and C of one sign: what follows it (backward: what is in front
    of it) is infinite with the definition's sign, the rest as without it, however many states a thread has room for."""
    s = make(1, length, d, n, 1, dtype, 51, state=True)
    rows = (torch.arange(d) * 7) % length
    at = (0, rows, torch.arange(d))
    for k in ("B", "C", "h", "x", "D", "dy", "dh"):
        s[k] = s[k].abs() + 0.01
    s["A"][:] = -0.1
    s["x"][at] = 0.5
    s["dy"][at] = 0.5
    s["z"] = s["z"].masked_fill(s["z"] == 0, 0.01)
    c = geometry(s, n, 1, 1)
    ref = reference(s, n, 1, 1, None, True, dtype)
    t = torch.arange(length)[None, :, None]
    behind = (t >= rows).expand(1, length, d)
    s["x"][at] = float("inf")
    y, h, saved = forward(lib, s, c, dtype, keep=True)
    y2, h2, _ = forward(lib, s, c, dtype)                          # a single token has a kernel of its own
    z = s["z"].double().cpu()
    for got in (y, y2):
        got = got.cpu()
        assert torch.equal(got.double()[behind], (float("inf") * z.sign())[behind])
        close(got[~behind], ref["y"][~behind], ref["y_slack"][~behind], "y")
    assert (h == float("inf")).all() and (h2 == float("inf")).all()
    dz = backward(lib, s, c, dtype, saved)["dz"].cpu()
    slope = 1 + z * torch.sigmoid(-z)
    assert torch.equal(dz.double()[behind], (float("inf") * slope.sign())[behind])
    close(dz[~behind], ref["dz"][~behind], ref["dz_slack"][~behind], "dz")
    # the gradients, without the gate
    s["x"][at] = 0.5
    s["z"] = None
    c = geometry(s, n, 1, 1)
    ref = reference(s, n, 1, 1, None, True, dtype)
    _, _, saved = forward(lib, s, c, dtype, keep=True)
    s["dy"][at] = float("inf")
    got = {k: v.cpu() for k, v in backward(lib, s, c, dtype, saved).items() if v is not None}
    front = (t <= rows).expand(1, length, d)
    assert (got["dx"][front] == float("inf")).all()
    close(got["dx"][~front], ref["dx"][~front], ref["dx_slack"][~front], "dx")
    for k in ("dA", "dD", "dh_in"):
        assert (got[k] == float("inf")).all(), k
    hit = torch.zeros(length, dtype=torch.bool)
    hit[rows] = True
    for k, inf in (("dC", hit), ("dB", torch.arange(length) <= int(rows.max()))):
        assert (got[k][:, inf] == float("inf")).all(), k
        close(got[k][:, ~inf], ref[k][:, ~inf], ref[k + "_slack"][:, ~inf], k)


def unmasked(s, n, groups, softplus, dtype):
    """Nothing overflows in the recurrence, so that no comparison with it is left out."""
    ref = reference(s, n, groups, softplus, None, True, dtype)
    assert all(torch.isfinite(v).all() for v in ref.values())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [1, 4, 6, 16, 24, 33, 64])
def test_step_sizes_given_as_they_are(lib, dtype, n):
    """softplus = 0 with positive dt: the states stay finite, so every value and gradient is compared; whole and split sequences."""
    for k, (batch, length, d, groups) in enumerate([(3, 17, 64, 2), (2, 33, 36, 3), (1, 300, 24, 1)]):
        s = make(batch, length, d, n, groups, dtype, 61 * n + k, state=k != 0, gate=k != 1, bias=False)
        s["dt"] = 0.3 * s["dt"].abs() + 0.01
        unmasked(s, n, groups, 0, dtype)
        check(lib, s, n, groups, 0, dtype, f"{dtype} n={n} {batch}x{length}x{d}/{groups}")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [4, 8, 12, 16, 32, 64])
@pytest.mark.parametrize("softplus", [0, 1])
def test_split_sequences_in_whole_packs(lib, dtype, n, softplus):
    """Split sequences whose every operand is aligned and whose blocks are full, two groups, two sequences: asynchronous copies in
    both passes and both directions, with states entering and gradients leaving."""
    lanes = 1
    while 4 * lanes < n:
        lanes *= 2
    d, length = 2 * (128 // lanes), 300
    s = make(2, length, d, n, 2, dtype, 67 + n, state=True, bias=softplus == 1)
    s["B"], s["C"] = s["B"].contiguous(), s["C"].contiguous()
    if not softplus:
        s["dt"] = 0.3 * s["dt"].abs() + 0.01
    assert all(s[k].data_ptr() % 16 == 0 and s[k].stride(1) * s[k].element_size() % 16 == 0 for k in ("x", "z", "dt", "B", "C", "dy"))
    unmasked(s, n, 2, softplus, dtype)
    c = check(lib, s, n, 2, softplus, dtype, f"{dtype} n={n} split")
    assert lib.rp_selective_scan_ws_bytes(C.byref(c), CODE[dtype], 0) > 0          # it is split


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,groups", [(16, 24, 1), (4, 130, 1), (8, 40, 2), (64, 9, 1), (6, 64, 1)])
def test_infinite_B_and_C_and_channels_that_leave_lanes_idle(lib, dtype, n, d, groups):
    """One infinite row of B, then of C, everything of one sign: dC (dB) is the infinity of the definition from (up to) that row on, also
    where a block has lanes for channels that are not there."""
    length, r = 45, 20
    s = make(1, length, d, n, groups, dtype, 71, state=True, gate=False)
    for k in ("B", "C", "h", "x", "D", "dy", "dh"):
        s[k] = s[k].abs() + 0.01
    s["A"][:] = -0.1
    c = geometry(s, n, groups, 1)
    for name, key, rows, wide in (("B", "dC", slice(r, None), slice(None, r)), ("C", "dB", slice(None, r + 1), slice(r + 1, None))):
        ref = reference(s, n, groups, 1, None, True, dtype)
        keep = s[name]
        s[name] = keep.clone()
        s[name][:, r] = float("inf")
        _, _, saved = forward(lib, s, c, dtype, keep=True)
        got = {k: v.cpu() for k, v in backward(lib, s, c, dtype, saved).items() if v is not None}
        assert (got[key][:, rows] == float("inf")).all(), key
        close(got[key][:, wide], ref[key][:, wide], ref[key + "_slack"][:, wide], key)
        s[name] = keep
