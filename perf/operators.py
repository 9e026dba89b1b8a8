"""The sequence operators of the library and how they are measured: the short causal convolution, the selective state
space scan and the gated block norm, each forward, as a training step (forward and backward) and for single tokens.

``own`` false: the plain form in elementary torch operations, float32 inside, rounded once at the end.
``own`` true: the library's entry points through the C ABI.  ``exact`` gives the same outputs in float64, computed step
by step from the definition.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"bf16": 3, "f16": 2, "f32": 0}
EPS = 1e-5


# --------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one token for each of 8 running requests: latency
        {"name": "conv_token", "op": "conv", "mode": "forward", "dtype": "bf16", "batch": 8, "len": 1, "channels": 2048, "width": 4,
         "state": True, "ragged": False},
        # prompts of a wide layer, x one half of a projection's output
        {"name": "conv_prompt", "op": "conv", "mode": "forward", "dtype": "bf16", "batch": 4, "len": 4096, "channels": 4096, "width": 4,
         "state": True, "ragged": True},
        # a training step with odd sizes
        {"name": "conv_train_odd", "op": "conv", "mode": "train", "dtype": "f16", "batch": 3, "len": 1999, "channels": 1531, "width": 3,
         "state": False, "ragged": False},
        # one token for each of 64 running requests: the state is what moves
        {"name": "scan_token", "op": "scan", "mode": "forward", "dtype": "bf16", "batch": 64, "len": 1, "channels": 4096, "states": 16,
         "groups": 1, "state": True, "gate": True, "ragged": False},
        # prompts of a wide layer
        {"name": "scan_prompt", "op": "scan", "mode": "forward", "dtype": "bf16", "batch": 2, "len": 4096, "channels": 4096, "states": 16,
         "groups": 1, "state": False, "gate": True, "ragged": False},
        # one long prompt of a narrow layer: few channels, so the length has to be split
        {"name": "scan_prompt_long", "op": "scan", "mode": "forward", "dtype": "f16", "batch": 1, "len": 16384, "channels": 512,
         "states": 16, "groups": 1, "state": True, "gate": True, "ragged": False},
        # a padded batch of prompts that continue from a state, float32, odd sizes
        {"name": "scan_prompt_ragged", "op": "scan", "mode": "forward", "dtype": "f32", "batch": 5, "len": 777, "channels": 650,
         "states": 24, "groups": 2, "state": True, "gate": False, "ragged": True},
        # a training step of a wide layer
        {"name": "scan_train", "op": "scan", "mode": "train", "dtype": "bf16", "batch": 2, "len": 2048, "channels": 4096, "states": 16,
         "groups": 1, "state": False, "gate": True, "ragged": False},
        # a training step with odd sizes, float32
        {"name": "scan_train_odd", "op": "scan", "mode": "train", "dtype": "f32", "batch": 3, "len": 509, "channels": 331, "states": 10,
         "groups": 1, "state": False, "gate": True, "ragged": False},
        # single tokens of 16 requests
        {"name": "norm_token", "op": "norm", "mode": "forward", "dtype": "bf16", "rows": 16, "channels": 2048, "gate": True},
        # prompts of a wide layer
        {"name": "norm_prompt", "op": "norm", "mode": "forward", "dtype": "bf16", "rows": 8192, "channels": 4096, "gate": True},
        # a training step with an odd row length
        {"name": "norm_train_odd", "op": "norm", "mode": "train", "dtype": "f16", "rows": 4001, "channels": 2999, "gate": True},
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["conv", "scan", "scan", "norm"])
    mode = rng.choice(["forward", "forward", "train"])
    case = {"op": op, "mode": mode, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op == "norm":
        channels = log_int(64, 8192)
        return {**case, "rows": log_int(1, min(32768, (1 << 25) // channels)), "channels": channels, "gate": rng.random() < 0.7}
    token = mode == "forward" and rng.random() < 0.25
    batch = log_int(1, 256) if token else log_int(1, 16)
    groups = rng.choice([1, 1, 1, 2, 4]) if op == "scan" else 1
    channels = groups * log_int(max(1, 64 // groups), 4096 // groups)
    state = token or (mode == "forward" and rng.random() < 0.5)
    ragged = mode == "forward" and not token and rng.random() < 0.4
    if op == "conv":
        most = (1 << 25) // (batch * channels)
        return {**case, "batch": batch, "len": 1 if token else log_int(2, max(2, min(16384, most))), "channels": channels,
                "width": rng.choice([2, 3, 4, 4, 4, 5, 8]), "state": state, "ragged": ragged}
    states = log_int(1, 64)
    most = (1 << 27) // (batch * channels * states)
    return {**case, "batch": batch, "len": 1 if token else log_int(2, max(2, min(16384, most))), "channels": channels,
            "states": states, "groups": groups, "state": state, "gate": rng.random() < 0.7, "ragged": ragged}


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    train = case["mode"] == "train"
    if case["op"] == "norm":
        n, d = case["rows"] * case["channels"], case["channels"]
        gate = 1 if case["gate"] else 0
        moved = e * (n * (2 + gate + 2) + 3 * d)                                    # u, (z), r in; out, y out
        if train:
            moved += e * (n * (2 + 2 + gate) + 3 * d)                               # dout, dy in; du, (dz), dr out
        return {"bytes": moved, "flops": n * (12 + 6 * gate) * (3 if train else 1)}
    rows = case["batch"] * case["len"]
    if case["op"] == "conv":
        n, d, w = rows * case["channels"], case["channels"], case["width"]
        moved = e * (2 * n + d * (w + 1))
        if case["state"]:
            moved += e * 2 * case["batch"] * (w - 1) * d
        if train:
            moved += e * (2 * n + d * (w + 1))
        return {"bytes": moved, "flops": n * (2 * w + 5) * (3 if train else 1)}
    n, d, s = rows * case["channels"], case["channels"], case["states"]
    gate = 1 if case["gate"] else 0
    bc = 2 * rows * case["groups"] * s
    moved = e * (n * (3 + gate) + bc) + 4 * (d * s + 2 * d)                         # x, dt, (z), B, C in; y out; A, D, dt_bias
    moved += 4 * case["batch"] * d * s * (2 if case["state"] else 0 if train else 1)
    if train:
        moved += e * (n * (3 + gate) + bc) + 4 * (d * s + 2 * d)                    # dy in; dx, ddt, (dz), dB, dC, dA, dD, ddt_bias out
    per_state = 8                                                                   # dt A, exp, (dt x) B, h = a h + ., y += C h
    return {"bytes": moved, "flops": n * s * per_state * (3 if train else 1) + n * 10}


# --------------------------------------------------------------------------------------------------- the inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, kind=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(kind)

    s = {"case": dict(case)}
    d = case["channels"]
    if case["op"] == "norm":
        rows = case["rows"]
        s["u"], s["r"] = normal(rows, d), normal(rows, d, scale=2.0)
        s["z"] = normal(rows, d) if case["gate"] else None
        s["w_after"], s["w_before"] = (1 + normal(d, scale=0.1).float()).to(dtype), (1 + normal(d, scale=0.1).float()).to(dtype)
        s["scale"] = normal(d, scale=0.3)
        if case["mode"] == "train":
            s["dout"], s["dy"] = normal(rows, d), normal(rows, d)
        return s
    batch, length = case["batch"], case["len"]
    s["x"], z = normal(batch, length, 2 * d).split(d, dim=2)                        # two halves of one projection's output
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(0, length + 1, (batch,), generator=gen, device="cuda", dtype=torch.int32)
        s["lengths"][0] = length
    if case["mode"] == "train":
        s["dy"] = normal(batch, length, d)
    if case["op"] == "conv":
        w = case["width"]
        s["w"], s["bias"] = normal(d, w, scale=w ** -0.5), normal(d, scale=0.1)
        s["state"] = normal(batch, w - 1, d) if case["state"] else None
        return s
    n, g = case["states"], case["groups"]
    s["z"] = z if case["gate"] else None
    # step sizes between 1e-3 and 1e-1 through the bias, as such layers are set up, and the token's own part on top
    step = torch.exp(torch.rand(d, generator=gen, device="cuda") * (math.log(0.1) - math.log(1e-3)) + math.log(1e-3))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    s["dt"] = normal(batch, length, d, scale=0.5)
    s["A"] = -torch.arange(1, n + 1, device="cuda").float() * torch.exp(0.1 * torch.randn(d, n, generator=gen, device="cuda"))
    s["D"] = 1 + 0.1 * torch.randn(d, generator=gen, device="cuda")
    rank = max(1, d // 16)
    _, s["B"], s["C"] = normal(batch, length, rank + 2 * g * n).split([rank, g * n, g * n], dim=2)   # slices of one projection
    s["h"] = normal(batch, d, n, kind=torch.float32) if case["state"] else None
    return s


# --------------------------------------------------------------------------------------------------- the plain form

def _silu_pair(z):
    """silu(z) and its derivative."""
    sig = torch.sigmoid(z)
    return z * sig, sig * (1 + z * (1 - sig))


def _rows_behind(lengths, length):
    return torch.arange(length, device=lengths.device)[None, :, None] >= lengths[:, None, None]


def _plain_conv(s, case):
    x, w, bias = s["x"].float(), s["w"].float(), s["bias"].float()
    width, dtype = case["width"], s["x"].dtype
    batch, length, d = x.shape
    first = s["state"].float() if s["state"] is not None else x.new_zeros(batch, width - 1, d)
    behind = None
    if s["lengths"] is not None:
        behind = _rows_behind(s["lengths"], length)
        x = x.masked_fill(behind, 0)
    xp = torch.cat([first, x], dim=1)
    taps = xp.unfold(1, width, 1)                                                   # [batch, length, d, width]
    pre = (taps * w).sum(-1) + bias
    y, slope = _silu_pair(pre)
    if behind is not None:
        y = y.masked_fill(behind, 0)
    out = {"y": y.to(dtype)}
    if case["state"]:
        last = s["lengths"].long() if s["lengths"] is not None else torch.full((batch,), length, device=x.device)
        at = (last[:, None] + torch.arange(width - 1, device=x.device))[:, :, None].expand(-1, -1, d)
        out["state"] = xp.gather(1, at).to(dtype)
    if case["mode"] == "train":
        dpre = s["dy"].float() * slope
        ahead = torch.nn.functional.pad(dpre, (0, 0, 0, width - 1)).unfold(1, width, 1)
        out["dx"] = (ahead * w.flip(1)).sum(-1).to(dtype)
        out["dw"] = (taps * dpre.unsqueeze(-1)).sum((0, 1)).to(dtype)
        out["dbias"] = dpre.sum((0, 1)).to(dtype)
    return out


def _linear_recurrence(a, b):
    """h[:, t] = a[:, t] h[:, t-1] + b[:, t] by doubling."""
    step = 1
    while step < b.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], dim=1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], dim=1)
        step *= 2
    return b


def _plain_scan(s, case):
    x, dt, A, D = s["x"].float(), s["dt"].float(), s["A"], s["D"]
    dtype, groups, n = s["x"].dtype, case["groups"], case["states"]
    batch, length, d = x.shape
    Bm = s["B"].float().reshape(batch, length, groups, 1, n)
    Cm = s["C"].float().reshape(batch, length, groups, 1, n)
    raw = dt + s["dt_bias"]
    delta = torch.nn.functional.softplus(raw)
    behind = None
    if s["lengths"] is not None:
        behind = _rows_behind(s["lengths"], length)
        x, delta = x.masked_fill(behind, 0), delta.masked_fill(behind, 0)
    by_group = lambda v: v.reshape(batch, length, groups, d // groups, -1)          # noqa: E731
    a = torch.exp(delta.unsqueeze(-1) * A)
    b = (by_group(delta * x) * Bm).reshape(batch, length, d, n)
    if s["h"] is not None:
        b[:, 0] += a[:, 0] * s["h"]
    h = _linear_recurrence(a, b)
    y = (by_group(h).reshape(batch, length, groups, d // groups, n) * Cm).sum(-1).reshape(batch, length, d) + D * x
    gate, slope = _silu_pair(s["z"].float()) if case["gate"] else (None, None)
    total = y * gate if case["gate"] else y
    if behind is not None:
        total = total.masked_fill(behind, 0)
    out = {"y": total.to(dtype)}
    if case["mode"] != "train":
        out["h"] = h[:, -1].contiguous()
        return out
    dy = s["dy"].float()
    if case["gate"]:
        out["dz"] = (dy * y * slope).to(dtype)
        dy = dy * gate
    dyc = (by_group(dy) * Cm).reshape(batch, length, d, n)
    following = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], dim=1)
    dh = _linear_recurrence(following.flip(1), dyc.flip(1)).flip(1)
    h_before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], dim=1)
    da = dh * h_before * a
    inner = (dh.reshape(batch, length, groups, d // groups, n) * Bm).sum(-1).reshape(batch, length, d)
    ddelta = (da * A).sum(-1) + inner * x
    ddt = ddelta * torch.sigmoid(raw)
    out["dx"] = (delta * inner + D * dy).to(dtype)
    out["ddt"] = ddt.to(dtype)
    out["dA"] = (da * delta.unsqueeze(-1)).sum((0, 1))
    out["dB"] = (dh * (delta * x).unsqueeze(-1)).reshape(batch, length, groups, d // groups, n).sum(3).reshape(batch, length, -1).to(dtype)
    out["dC"] = (h * dy.unsqueeze(-1)).reshape(batch, length, groups, d // groups, n).sum(3).reshape(batch, length, -1).to(dtype)
    out["dD"] = (dy * x).sum((0, 1))
    out["ddt_bias"] = ddt.sum((0, 1))
    return out


def _plain_norm(s, case):
    u, r, dtype = s["u"].float(), s["r"].float(), s["u"].dtype
    w_after, w_before, scale = s["w_after"].float(), s["w_before"].float(), s["scale"].float()
    gate, slope = _silu_pair(s["z"].float()) if case["gate"] else (None, None)
    v = u * gate if case["gate"] else u
    i1 = torch.rsqrt(v.square().mean(1, keepdim=True) + EPS)
    out = r + scale * (v * i1 * w_after)
    i2 = torch.rsqrt(out.square().mean(1, keepdim=True) + EPS)
    res = {"out": out.to(dtype), "y": (out * i2 * w_before).to(dtype)}
    if case["mode"] != "train":
        return res
    dout, dy = s["dout"].float(), s["dy"].float()
    res["dw_before"] = (dy * out * i2).sum(0).to(dtype)
    m = dy * w_before
    total = dout + i2 * (m - out * i2.square() * (m * out).mean(1, keepdim=True))
    res["dr"] = total.to(dtype)
    res["dscale"] = (total * v * i1 * w_after).sum(0).to(dtype)
    res["dw_after"] = (total * scale * v * i1).sum(0).to(dtype)
    m = total * scale * w_after
    dv = i1 * (m - v * i1.square() * (m * v).mean(1, keepdim=True))
    res["du"] = (dv * gate if case["gate"] else dv).to(dtype)
    if case["gate"]:
        res["dz"] = (dv * u * slope).to(dtype)
    return res


# --------------------------------------------------------------------------------------------------- the library

def _ptr(t):
    return None if t is None else t.data_ptr()


def _checked(rc):
    if rc != 0:
        raise RuntimeError("the library refused the call")


def _own_conv(s, case):
    import recpulse_b200 as rpb
    lib, code, stream = rpb.load(), CODES[case["dtype"]], torch.cuda.current_stream().cuda_stream
    x, w, bias, state = s["x"], s["w"], s["bias"], s["state"]
    batch, length, d = x.shape
    y = torch.empty(batch, length, d, dtype=x.dtype, device=x.device)
    c = rpb.RpbCausalConv(batch, length, d, case["width"], 1, x.stride(0), x.stride(1), length * d, d, length * d, d)
    out = {"y": y}
    if case["state"]:
        out["state"] = torch.empty_like(state)
    _checked(lib.rp_causal_conv_ex(y.data_ptr(), _ptr(out.get("state")), x.data_ptr(), w.data_ptr(), bias.data_ptr(), _ptr(state),
                                   _ptr(s["lengths"]), c, code, 0, stream))
    if case["mode"] == "train":
        dx, dw, dbias = torch.empty_like(y), torch.empty_like(w), torch.empty_like(bias)
        ws = torch.empty(lib.rp_causal_conv_ws_bytes(c, code), dtype=torch.uint8, device=x.device)
        _checked(lib.rp_causal_conv_grad_ex(dx.data_ptr(), dw.data_ptr(), dbias.data_ptr(), None, 0, s["dy"].data_ptr(), None,
                                            x.data_ptr(), w.data_ptr(), bias.data_ptr(), None, None, ws.data_ptr(), c, code, 0, stream))
        out.update(dx=dx, dw=dw, dbias=dbias)
    return out


def _own_scan(s, case):
    import recpulse_b200 as rpb
    lib, code, stream = rpb.load(), CODES[case["dtype"]], torch.cuda.current_stream().cuda_stream
    x, dt, Bm, Cm, z = s["x"], s["dt"], s["B"], s["C"], s["z"]
    A, D, dt_bias = s["A"], s["D"], s["dt_bias"]
    batch, length, d = x.shape
    n, gn = case["states"], case["groups"] * case["states"]
    new = lambda *shape, dtype=x.dtype: torch.empty(*shape, dtype=dtype, device=x.device)      # noqa: E731
    y = new(batch, length, d)
    zs = (z.stride(0), z.stride(1)) if z is not None else (0, 0)
    row, col = (length * d, d), (length * gn, gn)
    both = (length * 2 * d, 2 * d) if z is not None else row                        # dx and dz: the halves of one buffer
    c = rpb.RpbScan(batch, length, d, n, case["groups"], 1, x.stride(0), x.stride(1), dt.stride(0), dt.stride(1), Bm.stride(0), Bm.stride(1),
                    Cm.stride(0), Cm.stride(1), *zs, *row, *both, *row, *col, *col, *both)
    train = case["mode"] == "train"
    h = None if train else new(batch, d, n, dtype=torch.float32)
    saved = new(lib.rp_selective_scan_saved_elems(c, code), dtype=torch.float32) if train else None
    size = lib.rp_selective_scan_ws_bytes(c, code, 0)
    ws = new(size, dtype=torch.uint8) if size else None
    _checked(lib.rp_selective_scan_ex(y.data_ptr(), _ptr(h), _ptr(saved), x.data_ptr(), dt.data_ptr(), A.data_ptr(), Bm.data_ptr(), Cm.data_ptr(),
                                      D.data_ptr(), dt_bias.data_ptr(), _ptr(z), _ptr(s["h"]), _ptr(s["lengths"]), _ptr(ws), c, code, 0, stream))
    if not train:
        return {"y": y, "h": h}
    out = {"y": y}
    if z is not None:
        out["dx"], out["dz"] = new(batch, length, 2 * d).split(d, dim=2)
    else:
        out["dx"] = new(batch, length, d)
    out.update(ddt=new(batch, length, d), dA=torch.empty_like(A), dB=new(batch, length, gn), dC=new(batch, length, gn),
               dD=torch.empty_like(D), ddt_bias=torch.empty_like(dt_bias))
    ws = new(lib.rp_selective_scan_ws_bytes(c, code, 1), dtype=torch.uint8)
    _checked(lib.rp_selective_scan_grad_ex(out["dx"].data_ptr(), out["ddt"].data_ptr(), out["dA"].data_ptr(), out["dB"].data_ptr(),
                                           out["dC"].data_ptr(), out["dD"].data_ptr(), out["ddt_bias"].data_ptr(), _ptr(out.get("dz")), None, 0,
                                           s["dy"].data_ptr(), None, x.data_ptr(), dt.data_ptr(), A.data_ptr(), Bm.data_ptr(), Cm.data_ptr(),
                                           D.data_ptr(), dt_bias.data_ptr(), _ptr(z), None, saved.data_ptr(), ws.data_ptr(), c, code, 0, stream))
    return out


def _own_norm(s, case):
    import recpulse_b200 as rpb
    lib, code, stream = rpb.load(), CODES[case["dtype"]], torch.cuda.current_stream().cuda_stream
    u, z, r = s["u"], s["z"], s["r"]
    rows, d = u.shape
    c = rpb.RpbBlockNorm(rows, d, EPS, EPS, d, d, d, d, d, d, d, d)
    out = {"out": torch.empty_like(u), "y": torch.empty_like(u)}
    args = (u.data_ptr(), _ptr(z), s["w_after"].data_ptr(), s["scale"].data_ptr(), r.data_ptr(), s["w_before"].data_ptr())
    _checked(lib.rp_block_norm_ex(out["out"].data_ptr(), out["y"].data_ptr(), *args, c, code, 0, stream))
    if case["mode"] == "train":
        out.update(du=torch.empty_like(u), dr=torch.empty_like(u), dw_after=torch.empty_like(s["w_after"]),
                   dscale=torch.empty_like(s["scale"]), dw_before=torch.empty_like(s["w_before"]))
        if z is not None:
            out["dz"] = torch.empty_like(u)
        ws = torch.empty(lib.rp_block_norm_ws_bytes(c, code), dtype=torch.uint8, device=u.device)
        _checked(lib.rp_block_norm_grad_ex(out["du"].data_ptr(), _ptr(out.get("dz")), out["dr"].data_ptr(), out["dw_after"].data_ptr(),
                                           out["dscale"].data_ptr(), out["dw_before"].data_ptr(), 0, s["dout"].data_ptr(), s["dy"].data_ptr(),
                                           *args, ws.data_ptr(), c, code, 0, stream))
    return out


def run(state):
    case = state["case"]
    if own:
        return {"conv": _own_conv, "scan": _own_scan, "norm": _own_norm}[case["op"]](state, case)
    return {"conv": _plain_conv, "scan": _plain_scan, "norm": _plain_norm}[case["op"]](state, case)


# --------------------------------------------------------------------------------------------------- in 64 bits

def _exact_conv(s, case):
    x, w, bias = s["x"].double(), s["w"].double(), s["bias"].double()
    batch, length, d = x.shape
    width = case["width"]
    ends = s["lengths"].tolist() if s["lengths"] is not None else [length] * batch
    y, state = torch.zeros_like(x), x.new_zeros(batch, width - 1, d)
    dx, dw, dbias = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(bias)
    for b, end in enumerate(ends):
        line = torch.cat([s["state"][b].double() if s["state"] is not None else x.new_zeros(width - 1, d), x[b, :end]])
        state[b] = line[end:]
        pre = bias.expand(end, d).clone()
        for j in range(width):
            pre += w[:, j] * line[j:j + end]
        y[b, :end] = pre / (1 + torch.exp(-pre))
        if case["mode"] == "train":
            sig = 1 / (1 + torch.exp(-pre))
            dpre = s["dy"][b].double() * (sig + pre * sig * (1 - sig))
            back = torch.zeros_like(line)
            for j in range(width):
                back[j:j + end] += w[:, j] * dpre
                dw[:, j] += (dpre * line[j:j + end]).sum(0)
            dx[b], dbias = back[width - 1:], dbias + dpre.sum(0)
    out = {"y": y}
    if case["state"]:
        out["state"] = state
    if case["mode"] == "train":
        out.update(dx=dx, dw=dw, dbias=dbias)
    return out


def _exact_scan(s, case):
    x, A, D = s["x"].double(), s["A"].double(), s["D"].double()
    batch, length, d = x.shape
    n, groups = case["states"], case["groups"]
    raw = s["dt"].double() + s["dt_bias"].double()
    delta = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))
    spread = lambda v, t: v[:, t].double().reshape(batch, groups, n).repeat_interleave(d // groups, dim=1)      # noqa: E731
    ends = s["lengths"][:, None, None] if s["lengths"] is not None else None
    h = s["h"].double() if s["h"] is not None else x.new_zeros(batch, d, n)
    train = case["mode"] == "train"
    past, core = [h], torch.zeros_like(x)
    for t in range(length):
        step = delta[:, t, :, None]
        nxt = torch.exp(step * A) * h + step * x[:, t, :, None] * spread(s["B"], t)
        h = nxt if ends is None else torch.where(t < ends, nxt, h)
        core[:, t] = (h * spread(s["C"], t)).sum(-1) + D * x[:, t]
        if train:
            past.append(h)
    z = s["z"].double() if case["gate"] else None
    sig = 1 / (1 + torch.exp(-z)) if case["gate"] else None
    y = core * z * sig if case["gate"] else core.clone()
    if ends is not None:
        y *= torch.arange(length, device=x.device)[None, :, None] < ends
    if not train:
        return {"y": y, "h": h}
    dy = s["dy"].double()
    out = {"y": y}
    if case["gate"]:
        out["dz"] = dy * core * (sig + z * sig * (1 - sig))
        dy = dy * z * sig
    dx, ddelta, dA = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(A)
    dB, dC = (x.new_zeros(batch, length, groups * n) for _ in range(2))
    dh = torch.zeros_like(h)
    for t in range(length - 1, -1, -1):
        step, a = delta[:, t, :, None], torch.exp(delta[:, t, :, None] * A)
        dh = dh + dy[:, t, :, None] * spread(s["C"], t)
        dC[:, t] = (dy[:, t, :, None] * past[t + 1]).reshape(batch, groups, d // groups, n).sum(2).reshape(batch, -1)
        dB[:, t] = (dh * step * x[:, t, :, None]).reshape(batch, groups, d // groups, n).sum(2).reshape(batch, -1)
        inner = (dh * spread(s["B"], t)).sum(-1)
        decay = dh * past[t] * a
        ddelta[:, t] = (decay * A).sum(-1) + inner * x[:, t]
        dx[:, t] = delta[:, t] * inner + D * dy[:, t]
        dA += (decay * step).sum(0)
        dh = dh * a
    ddt = ddelta / (1 + torch.exp(-raw))
    out.update(dx=dx, ddt=ddt, dA=dA, dB=dB, dC=dC, dD=(dy * x).sum((0, 1)), ddt_bias=ddt.sum((0, 1)))
    return out


def _exact_norm(s, case):
    """The gradients from the Jacobian of v / |v|, with |v| as the root of the mean square."""
    u, r = s["u"].double(), s["r"].double()
    wa, wb, scale = s["w_after"].double(), s["w_before"].double(), s["scale"].double()
    d = u.shape[1]
    z = s["z"].double() if case["gate"] else None
    sig = 1 / (1 + torch.exp(-z)) if case["gate"] else None
    v = u * z * sig if case["gate"] else u
    size1 = ((v * v).sum(1, keepdim=True) / d + EPS).sqrt()
    unit1 = v / size1
    out = r + scale * wa * unit1
    size2 = ((out * out).sum(1, keepdim=True) / d + EPS).sqrt()
    unit2 = out / size2
    res = {"out": out, "y": unit2 * wb}
    if case["mode"] != "train":
        return res
    back = lambda g, unit, size: (g - unit * (g * unit).sum(1, keepdim=True) / d) / size       # noqa: E731
    dy = s["dy"].double()
    total = s["dout"].double() + back(dy * wb, unit2, size2)
    dv = back(total * scale * wa, unit1, size1)
    res.update(dr=total, dw_before=(dy * unit2).sum(0), dscale=(total * wa * unit1).sum(0), dw_after=(total * scale * unit1).sum(0))
    res["du"] = dv * z * sig if case["gate"] else dv
    if case["gate"]:
        res["dz"] = dv * u * (sig + z * sig * (1 - sig))
    return res


def exact(case, seed):
    s = prepare(case, seed)
    return {"conv": _exact_conv, "scan": _exact_scan, "norm": _exact_norm}[case["op"]](s, case)
