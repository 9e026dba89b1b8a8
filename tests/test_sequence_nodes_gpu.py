"""The operators along a sequence as nodes: each against the float64 formulas (through torch's own gradients of them), together as
one recurrent block with the matmul nodes, accumulation, views, refusals, stream order and a captured step."""
import ctypes as C

import numpy as np
import pytest
import torch

import recpulse_b200 as rpb
from oracle import oracle as O
from helpers import CODE, f64, rand_operand

pytestmark = pytest.mark.gpu
EPS = 1e-5
# A gradient of these chains sums at most about 1e3 products and passes a dozen steps: 1e3 half-steps of the type that holds the
# sums bound the relative error in norm (float32: 6e-5, float64: 1.1e-13, ten times that for the conditioning of the norms), and
# every tensor that a 16-bit chain stores adds half a step of its own (bfloat16 2^-9 in norm at most, twelve tensors).
TOL = {"float32": 6e-5, "float64": 1.1e-12, "bfloat16": 12 * 2.0 ** -9, "float16": 12 * 2.0 ** -12}


@pytest.fixture(scope="module")
def lib():
    lib = rpb.load()
    yield lib
    lib.rpb_node_stream(None, 1)
    assert lib.rpb_device_status(0) == 0


def T(bits, dtype, grad=False):
    return rpb.Tensor.from_numpy(np.ascontiguousarray(bits), dtype=dtype, requires_grad=grad)


def rel(got, want):
    return float(np.linalg.norm(got - want) / (np.linalg.norm(want) or 1.0))


def conv64(x, w, b, silu=True):
    width = w.shape[1]
    xp = torch.nn.functional.pad(x, (0, 0, width - 1, 0))
    pre = sum(w[:, j] * xp[:, j:j + x.shape[1]] for j in range(width))
    pre = pre if b is None else pre + b
    return torch.nn.functional.silu(pre) if silu else pre


def scan64(x, dt, A, B, Cm, D, bias, z, softplus=True):
    batch, length, d = x.shape
    n = A.shape[1]
    g = B.shape[2] // n
    delta = dt if bias is None else dt + bias
    delta = torch.nn.functional.softplus(delta) if softplus else delta
    h, ys = torch.zeros(batch, d, n, dtype=x.dtype), []
    rep = lambda v, t: v[:, t].reshape(batch, g, n).repeat_interleave(d // g, dim=1)      # noqa: E731
    for t in range(length):
        h = torch.exp(delta[:, t, :, None] * A) * h + (delta * x)[:, t, :, None] * rep(B, t)
        ys.append((h * rep(Cm, t)).sum(-1))
    y = torch.stack(ys, 1)
    y = y if D is None else y + D * x
    return y if z is None else y * torch.nn.functional.silu(z)


def norm64(u, z, w, s, r):
    v = u if z is None else u * torch.nn.functional.silu(z)
    v = v if w is None else v / torch.sqrt((v * v).mean(-1, keepdim=True) + float(np.float32(EPS))) * w
    v = v if s is None else v * s
    return v if r is None else v + r


def leaf(a):
    return torch.tensor(a, dtype=torch.float64, requires_grad=True)


def acc(dtype):
    return "float64" if dtype == "float64" else "float32"


def check(node, leaves, value, grad, dtype):
    """`leaves`: (Tensor, torch leaf) pairs; runs the node's backward and compares everything."""
    assert rel(f64(node.to_numpy(), dtype), value.detach().numpy()) <= TOL[dtype]
    node.backward(T(grad, dtype))
    value.backward(torch.tensor(f64(grad, dtype)))
    for k, (t, l) in enumerate(leaves):
        assert rel(f64(t.grad.to_numpy(), t.dtype), l.grad.numpy()) <= TOL[dtype], k


@pytest.mark.parametrize("dtype", ["float32", "float64", "float16", "bfloat16"])
def test_nodes_against_the_formulas(lib, dtype):
    rng = np.random.default_rng(5)
    batch, length, d, n, g, width = 2, 19, 24, 6, 2, 3
    r = lambda *s, scale=1.0, dt=dtype: rand_operand(rng, s, dt, scale=scale)       # noqa: E731
    x, w, b, gy = r(batch, length, d), r(d, width), r(d), r(batch, length, d)
    for bias in (b, None):
        X, W, Bi = T(x, dtype, True), T(w, dtype, True), T(bias, dtype, True) if bias is not None else None
        lx, lw, lb = leaf(f64(x, dtype)), leaf(f64(w, dtype)), leaf(f64(bias, dtype)) if bias is not None else None
        check(X.op_causal_conv(W, Bi), [(X, lx), (W, lw)] + ([(Bi, lb)] if bias is not None else []), conv64(lx, lw, lb), gy, dtype)
    a = acc(dtype)
    A = -np.abs(rng.standard_normal((d, n))) - 0.1
    A, D, db = (v.astype(np.float64 if a == "float64" else np.float32) for v in (A, rng.standard_normal(d), rng.standard_normal(d)))
    dt, Bm, Cm, z = r(batch, length, d), r(batch, length, g * n), r(batch, length, g * n), r(batch, length, d)
    for parts in ((D, db, z), (None, None, None), (D, None, z)):
        args = [(x, dtype), (dt, dtype), (A, a), (Bm, dtype), (Cm, dtype)] + [(v, dtype if v is z else a) for v in parts if v is not None]
        ts = [T(v, k, True) for v, k in args]
        ls = [leaf(f64(v, k)) for v, k in args]
        opt, lopt, i = [], [], 5
        for v in parts:
            opt.append(ts[i] if v is not None else None); lopt.append(ls[i] if v is not None else None)
            i += v is not None
        node = ts[0].op_selective_scan(*ts[1:5], *opt)
        check(node, list(zip(ts, ls)), scan64(*ls[:5], *lopt), gy, dtype)
    s, rr = r(d), r(batch, length, d)
    for use in ((1, 1, 1, 1), (0, 1, 0, 0), (1, 0, 0, 1), (0, 0, 1, 1)):
        args = [x] + [v for v, on in zip((z, w[:, 0].copy(), s, rr), use) if on]
        ts, ls = [T(v, dtype, True) for v in args], [leaf(f64(v, dtype)) for v in args]
        it, lt = iter(ts[1:]), iter(ls[1:])
        opt, lopt = [next(it) if on else None for on in use], [next(lt) if on else None for on in use]
        node = ts[0].op_gated_norm(opt[0], opt[1], opt[2], opt[3], EPS)
        check(node, list(zip(ts, ls)), norm64(ls[0], *lopt), gy, dtype)
    X, W, lx, lw = T(x, dtype, True), T(s, dtype, True), leaf(f64(x, dtype)), leaf(f64(s, dtype))
    check(X.op_rms_norm(W, EPS), [(X, lx), (W, lw)], norm64(lx, None, lw, None, None), gy, dtype)


def block(params, x, dtype):
    """x + scale * (gated norm of a scan block), from nodes; returns the output and a function that runs all backwards."""
    batch, length, width = x.shape
    d, n, rank = params["A"].shape[0], params["A"].shape[1], params["w_dt"].shape[0]
    y0 = x.op_rms_norm(params["w_in_norm"], EPS)
    xz = y0.op_linear(params["w_in"], params["b_in"])
    xs, z = (xz.as_strided([batch, length, d], [length * 2 * d, 2 * d, 1], off) for off in (0, d))
    u = xs.op_causal_conv(params["w_conv"], params["b_conv"])
    low = u.op_matmul(params["w_x"])
    cols = rank + 2 * n
    cut = lambda off, w: low.as_strided([batch, length, w], [length * cols, cols, 1], off)       # noqa: E731
    low_dt, Bm, Cm = cut(0, rank), cut(rank, n), cut(rank + n, n)
    dt = low_dt.op_matmul(params["w_dt"])
    y = u.op_selective_scan(dt, params["A"], Bm, Cm, params["D"], params["dt_bias"], None)
    normed = y.op_gated_norm(z, params["w_norm"], None, None, EPS)
    proj = normed.op_matmul(params["w_out"])
    out = proj.op_gated_norm(None, None, params["scale"], x, EPS)

    def run_backward(grad):
        out.backward(grad)
        proj.backward(proj.grad)
        normed.backward(normed.grad)
        y.backward(y.grad)
        dt.backward(dt.grad)
        join = lambda parts: T(np.concatenate([p.grad.to_numpy() for p in parts], axis=2), dtype)      # noqa: E731
        low.backward(join([low_dt, Bm, Cm]))          # adds to what the scan left in u's gradient
        u.backward(u.grad)
        xz.backward(join([xs, z]))
        y0.backward(y0.grad)                          # adds to the residual's gradient of x

    return out, run_backward


def block64(p, x):
    d, n, rank = p["A"].shape[0], p["A"].shape[1], p["w_dt"].shape[0]
    xz = norm64(x, None, p["w_in_norm"], None, None) @ p["w_in"] + p["b_in"]
    u = conv64(xz[..., :d], p["w_conv"], p["b_conv"])
    low = u @ p["w_x"]
    y = scan64(u, low[..., :rank] @ p["w_dt"], p["A"], low[..., rank:rank + n], low[..., rank + n:], p["D"], p["dt_bias"], None)
    return x + p["scale"] * (norm64(y, xz[..., d:], p["w_norm"], None, None) @ p["w_out"])


def block_params(rng, dtype, width=32, d=48, n=8, rank=4):
    r = lambda *s, scale=1.0: (rand_operand(rng, s, dtype, scale=scale), dtype)      # noqa: E731
    a = acc(dtype)
    plain = lambda v: (v.astype(np.float64 if a == "float64" else np.float32), a)    # noqa: E731
    return {"w_in_norm": r(width), "w_in": r(width, 2 * d, scale=width ** -0.5), "b_in": r(2 * d, scale=0.1), "w_conv": r(d, 4, scale=0.5), "b_conv": r(d, scale=0.1),
            "w_x": r(d, rank + 2 * n, scale=d ** -0.5), "w_dt": r(rank, d, scale=rank ** -0.5), "A": plain(-np.arange(1, n + 1)[None, :] * np.ones((d, 1))),
            "D": plain(np.ones(d)), "dt_bias": plain(rng.uniform(-4, -1, d)), "w_norm": r(d), "w_out": r(d, width, scale=d ** -0.5), "scale": r(width)}


@pytest.mark.parametrize("dtype", ["float32", "float64", "bfloat16"])
def test_one_recurrent_block_trains_through_the_nodes(lib, dtype):
    """Norm, projection, convolution, low-rank step sizes, scan, gated norm, projection and the scaled residual: values and the
    gradients of every weight and of the input."""
    rng = np.random.default_rng(9)
    batch, length, width = 3, 21, 32
    params = block_params(rng, dtype)
    x = rand_operand(rng, (batch, length, width), dtype)
    g = rand_operand(rng, (batch, length, width), dtype)
    ps = {k: T(v, dt, True) for k, (v, dt) in params.items()}
    X = T(x, dtype, True)
    out, run_backward = block(ps, X, dtype)
    run_backward(T(g, dtype))
    ls, lx = {k: leaf(f64(v, dt)) for k, (v, dt) in params.items()}, leaf(f64(x, dtype))
    want = block64(ls, lx)
    want.backward(torch.tensor(f64(g, dtype)))
    assert rel(f64(out.to_numpy(), dtype), want.detach().numpy()) <= TOL[dtype]
    assert rel(f64(X.grad.to_numpy(), dtype), lx.grad.numpy()) <= TOL[dtype]
    for k in ps:
        assert rel(f64(ps[k].grad.to_numpy(), ps[k].dtype), ls[k].grad.numpy()) <= TOL[dtype], k
    # a second step adds to every gradient
    first = {k: f64(t.grad.to_numpy(), t.dtype) for k, t in ps.items()}
    out, run_backward = block(ps, X, dtype)
    run_backward(T(g, dtype))
    for k in ps:
        assert rel(f64(ps[k].grad.to_numpy(), ps[k].dtype), 2 * first[k]) <= TOL[dtype], k


def test_nodes_refuse(lib):
    rng = np.random.default_rng(3)
    dtype = "float32"
    r = lambda *s, dt=dtype, grad=False: T(rand_operand(rng, s, dt), dt, grad)       # noqa: E731
    x, w = r(2, 5, 8), r(8, 4)
    for bad in (lambda: r(2, 5).op_causal_conv(w), lambda: x.op_causal_conv(r(7, 4)), lambda: x.op_causal_conv(r(8, 9)),
                lambda: x.op_causal_conv(w, r(7)), lambda: x.op_causal_conv(r(8, 4, dt="float64")), lambda: x.transpose(1, 2).op_causal_conv(r(5, 2))):
        with pytest.raises(RuntimeError):
            bad()
    dt, A, B, Cm = r(2, 5, 8), r(8, 4), r(2, 5, 8), r(2, 5, 8)
    x.op_selective_scan(dt, A, B, Cm)
    same = r(2, 5, 8, grad=True)
    for bad in (lambda: x.op_selective_scan(r(2, 4, 8), A, B, Cm), lambda: x.op_selective_scan(dt, r(7, 4), B, Cm), lambda: x.op_selective_scan(dt, r(8, 3), B, Cm),
                lambda: x.op_selective_scan(dt, A, B, r(2, 5, 4)), lambda: x.op_selective_scan(dt, r(8, 4, dt="float64"), B, Cm),
                lambda: x.op_selective_scan(dt, A, r(2, 5, 12), r(2, 5, 12)), lambda: x.op_selective_scan(dt, A, B, Cm, r(7)),
                lambda: same.op_selective_scan(dt, A, B, Cm, None, None, same)):
        with pytest.raises(RuntimeError):
            bad()
    for bad in (lambda: x.op_rms_norm(r(7)), lambda: x.op_gated_norm(r(2, 5, 7), None), lambda: same.op_gated_norm(same, None), lambda: x.op_rms_norm(r(8, dt="float64"))):
        with pytest.raises(RuntimeError):
            bad()
    # a wrong upstream gradient leaves the gradients alone
    s = r(2, 5, 8, grad=True)
    y = s.op_causal_conv(w)
    y.backward(r(2, 5, 7))
    assert s.grad is None


def test_a_block_replayed_from_a_graph(lib):
    """The capture recipe of the matmul nodes for one forward and backward of all four new nodes, replayed with new inputs; a
    second graph of the same leaves alive beside it shares no workspace with the first."""
    dtype, batch, length, d, n = "float32", 2, 150, 16, 4
    rng = np.random.default_rng(21)
    r = lambda *s, grad=False: T(rand_operand(rng, s, dtype), dtype, grad)       # noqa: E731
    x, w, dt, B, Cm, z = r(batch, length, d, grad=True), r(d, 4, grad=True), r(batch, length, d), r(batch, length, n), r(batch, length, n), r(batch, length, d)
    A = T((-np.abs(rng.standard_normal((d, n))) - 0.1).astype(np.float32), dtype, True)
    s, g = r(d, grad=True), r(batch, length, d)

    def step():
        u = x.op_causal_conv(w)
        y = u.op_selective_scan(dt, A, B, Cm)
        o = y.op_gated_norm(z, s)
        o.backward(g); y.backward(y.grad); u.backward(u.grad)
        return o

    step()
    for t in (x, w, A, s):
        t.zero_grad()
    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        lib.rpb_node_stream(C.c_void_p(side.cuda_stream), 0)
        try:
            with torch.cuda.graph(graph, stream=side):
                o = step()
                grads = [t.grad for t in (x, w, A, s)]
        finally:
            lib.rpb_node_stream(None, 1)
        graphs.append((graph, o, grads))
        for t in (x, w, A, s):
            t.zero_grad()
    for trial, (graph, o, grads) in enumerate(graphs + graphs):
        bits = rand_operand(rng, (batch, length, d), dtype)
        x.copy_from_numpy(bits)
        graph.replay()
        torch.cuda.synchronize()
        ls = [leaf(f64(t.to_numpy(), dtype)) for t in (x, w, A, s)]
        u = conv64(ls[0], ls[1], None)
        want = norm64(scan64(u, *(torch.tensor(f64(t.to_numpy(), dtype)) if t is not A else ls[2] for t in (dt, A, B, Cm)), None, None, None),
                      torch.tensor(f64(z.to_numpy(), dtype)), ls[3], None, None)
        want.backward(torch.tensor(f64(g.to_numpy(), dtype)))
        assert rel(f64(o.to_numpy(), dtype), want.detach().numpy()) <= TOL[dtype], trial
        for got, l in zip(grads, ls):
            assert rel(f64(got.to_numpy(), dtype), l.grad.numpy()) <= TOL[dtype], trial


@pytest.mark.parametrize("shape,strides", [((4, 1, 8), (40, 8, 1)), ((4, 1, 5, 8), (40, 3, 8, 1)), ((1, 5, 8), (7, 8, 1)), ((2, 3, 1, 8), (48, 16, 1, 1)),
                                           ((1, 1, 8), (3, 5, 1)), ((4, 5, 8), (0, 0, 1))])
def test_norm_nodes_take_rows_at_one_distance(lib, shape, strides):
    """Dimensions of size 1 may have any stride; the upstream gradient likewise."""
    rng = np.random.default_rng(11)
    dtype, size = "float32", 1 + sum((n - 1) * s for n, s in zip(shape, strides))
    base, w = rand_operand(rng, (size,), dtype), rand_operand(rng, (8,), dtype)
    cut = lambda a: np.lib.stride_tricks.as_strided(a, shape, [4 * s for s in strides])       # noqa: E731
    u, lu = T(base, dtype, True).as_strided(shape, strides), leaf(f64(cut(base), dtype).copy())
    W, lw = T(w, dtype, True), leaf(f64(w, dtype))
    node, value = u.op_rms_norm(W, EPS), norm64(lu, None, lw, None, None)
    g = rand_operand(rng, (size,), dtype)
    assert rel(f64(node.to_numpy(), dtype), value.detach().numpy()) <= TOL[dtype]
    node.backward(T(g, dtype).as_strided(shape, strides))
    value.backward(torch.tensor(f64(cut(g), dtype).copy()))
    assert rel(f64(u.grad.to_numpy(), dtype), lu.grad.numpy()) <= TOL[dtype]
    assert rel(f64(W.grad.to_numpy(), dtype), lw.grad.numpy()) <= TOL[dtype]


def test_norm_nodes_refuse_rows_at_several_distances(lib):
    rng = np.random.default_rng(12)
    base, w = T(rand_operand(rng, (4, 1, 10, 8), "float32"), "float32"), T(rand_operand(rng, (8,), "float32"), "float32")
    with pytest.raises(RuntimeError):
        base.as_strided((4, 1, 5, 8), (80, 80, 8, 1)).op_rms_norm(w)
