/*
 * Short causal convolution along a sequence, one filter per channel, with its SiLU and its gradients:
 *   pre[b,t,d] = bias[d] + sum over j < width of w[d,j] * xp[b,t+j,d],   y = pre or pre / (1 + exp(-pre))
 * where xp is x behind width-1 earlier rows (the state of the sequence, or zeros).
 */
#include "seq_common.cuh"

namespace rpb_conv1d {

using namespace rpb_seq;

struct Args {
    int batch, len, channels, silu;
    long long x_batch, x_row, y_batch, y_row, dx_batch, dx_row;
    int run, runs;          /* rows per thread, and such runs per sequence */
    int n_vec;              /* packs of channels */
    bool vec_x, vec_y, vec_dx, vec_p;       /* whole packs may be moved: x, y (dy), dx, packed operands (state, bias) */
};

template <typename T> struct Width { static constexpr int fwd = 16 / sizeof(T), bwd = sizeof(T) == 2 ? 4 : 16 / sizeof(T); };

__device__ __forceinline__ int row_end(const int* lengths, int b, int len) {
    if (!lengths) return len;
    const int n = lengths[b];
    return n < 0 ? 0 : n > len ? len : n;
}

template <typename A> __device__ __forceinline__ A act(A pre, int silu) { return silu ? pre * logistic(pre) : pre; }
template <typename A> __device__ __forceinline__ A act_slope(A pre, int silu) {
    if (!silu) return A(1);
    const A s = logistic(pre);
    return s * (A(1) + pre * (A(1) - s));
}

/* w[V][W] and bias[V] of the channels from d0 on, 0 behind the last one */
template <typename T, int W, int V, typename A>
__device__ __forceinline__ void load_taps(A (&w)[V][W], A (&bias)[V], const T* wt, const T* bt, int d0, int channels) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const bool on = d0 + i < channels;
#pragma unroll
        for (int j = 0; j < W; ++j) w[i][j] = on ? up(wt[(long long)(d0 + i) * W + j]) : A(0);
        bias[i] = on && bt ? up(bt[d0 + i]) : A(0);
    }
}

/* Row p of xp before row 0 of x: row p + W - 1 of the sequence's state, zeros without one. */
template <typename T, int W, int V>
__device__ __forceinline__ Pack<T, V> state_row(const T* state, int b, int p, int d0, const Args& a) {
    if (!state) return zero_pack<T, V>();
    return load_pack<T, V>(state + ((long long)b * (W - 1) + p + W - 1) * a.channels + d0, a.channels - d0, a.vec_p);
}

/* One thread: V channels (16 bytes) of `run` consecutive rows, the last W - 1 rows in registers, so that x is read
 * once but for W - 1 rows in front of each run. */
template <typename T, int W>
__global__ void __launch_bounds__(128) forward_kernel(T* __restrict__ y, T* state_out, const T* __restrict__ x, const T* __restrict__ wt,
                                                      const T* __restrict__ bt, const T* state_in, const int* __restrict__ lengths, Args a) {
    typedef typename AccOf<T>::type A;
    constexpr int V = Width<T>::fwd, H = W - 1, U = 4;
    rpb_pdl_trigger();
    rpb_pdl_wait();
    const long long item = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const long long seq = item / a.n_vec;
    if (seq >= (long long)a.batch * a.runs) return;
    const int d0 = (int)(item - seq * a.n_vec) * V, valid = a.channels - d0;
    const int b = (int)(seq / a.runs), t0 = (int)(seq - (long long)b * a.runs) * a.run;
    const int t1 = t0 + a.run < a.len ? t0 + a.run : a.len, end = row_end(lengths, b, a.len);
    const T* xs = x + b * a.x_batch + d0;
    T* ys = y + b * a.y_batch + d0;

    A w[V][W], bias[V], win[W][V];          /* win[j]: row t - H + j */
    load_taps<T, W, V>(w, bias, wt, bt, d0, a.channels);
#pragma unroll
    for (int j = 0; j < H; ++j) {
        const int p = t0 - H + j;
        const Pack<T, V> r = p < 0 ? state_row<T, W, V>(state_in, b, p, d0, a)
                                   : p < end ? load_pack<T, V>(xs + p * a.x_row, valid, a.vec_x) : zero_pack<T, V>();
#pragma unroll
        for (int i = 0; i < V; ++i) win[j][i] = up(r.v[i]);
    }
    if (state_out && t0 == 0) {
        /* the last W - 1 rows of xp; all read before the first is written: state_out may be state_in */
        Pack<T, V> last[H > 0 ? H : 1];
#pragma unroll
        for (int j = 0; j < H; ++j) {
            const int p = end - H + j;
            last[j] = p < 0 ? state_row<T, W, V>(state_in, b, p, d0, a) : load_pack<T, V>(xs + p * a.x_row, valid, a.vec_x);
        }
#pragma unroll
        for (int j = 0; j < H; ++j) store_pack<T, V>(state_out + ((long long)b * H + j) * a.channels + d0, last[j], valid, a.vec_p);
    }
    for (int t = t0; t < t1; t += U) {
        Pack<T, V> rows[U];
#pragma unroll
        for (int k = 0; k < U; ++k)
            rows[k] = t + k < t1 && t + k < end ? load_pack<T, V>(xs + (t + k) * a.x_row, valid, a.vec_x) : zero_pack<T, V>();
#pragma unroll
        for (int k = 0; k < U; ++k) {
            if (t + k >= t1) break;
            Pack<T, V> o = zero_pack<T, V>();
#pragma unroll
            for (int i = 0; i < V; ++i) win[H][i] = up(rows[k].v[i]);
            if (t + k < end) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    A pre = bias[i];
#pragma unroll
                    for (int j = 0; j < W; ++j) pre += w[i][j] * win[j][i];
                    o.v[i] = down<T>(act(pre, a.silu));
                }
            }
            store_pack<T, V>(ys + (t + k) * a.y_row, o, valid, a.vec_y);
#pragma unroll
            for (int j = 0; j < H; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) win[j][i] = win[j + 1][i];
        }
    }
}

/* With dpre = dy act'(pre), 0 outside the sequence:
 *   dxp[p] = sum over j of w[j] dpre[p - j],   dw[j] = sum over t of dpre[t] xp[t + j],   dbias = sum of dpre.
 * A thread walks its rows upwards and W - 1 rows further, computes dpre of each row again from x and emits the gradient
 * of the row W - 1 behind; the run that begins a sequence emits the state's gradient in the same way.  The filter's
 * gradients of a block's four runs are added in shared memory and written as one part; sum_parts adds the parts. */
template <typename T, int W>
__global__ void __launch_bounds__(128) backward_kernel(T* dx, T* dstate_in, typename AccOf<T>::type* __restrict__ parts, int acc_dx,
                                                       const T* __restrict__ dy, const T* __restrict__ dstate_out, const T* __restrict__ x,
                                                       const T* __restrict__ wt, const T* __restrict__ bt, const T* __restrict__ state_in,
                                                       const int* __restrict__ lengths, Args a, int vec_blocks) {
    typedef typename AccOf<T>::type A;
    constexpr int V = Width<T>::bwd, H = W - 1;
    __shared__ A red[4][W + 1][32 * V + 1];
    rpb_pdl_trigger();
    rpb_pdl_wait();
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const long long group = blockIdx.x / vec_blocks;
    const int d0 = ((int)(blockIdx.x - group * vec_blocks) * 32 + tx) * V, valid = a.channels - d0;
    const long long seq = group * 4 + ty;
    A dw[V][W], db[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        db[i] = 0;
#pragma unroll
        for (int j = 0; j < W; ++j) dw[i][j] = 0;
    }
    if (valid > 0 && seq < (long long)a.batch * a.runs) {
        const int b = (int)(seq / a.runs), t0 = (int)(seq - (long long)b * a.runs) * a.run;
        const int t1 = t0 + a.run < a.len ? t0 + a.run : a.len, end = row_end(lengths, b, a.len);
        const T* xs = x + b * a.x_batch + d0;
        const T* gs = dy + b * a.y_batch + d0;
        T* ds = dx ? dx + b * a.dx_batch + d0 : nullptr;
        A w[V][W], bias[V], win[W][V], dp[W][V];        /* dp[j]: dpre of row s - H + j */
        load_taps<T, W, V>(w, bias, wt, bt, d0, a.channels);
#pragma unroll
        for (int j = 0; j < H; ++j) {
            const int p = t0 - H + j;
            const Pack<T, V> r = p < 0 ? state_row<T, W, V>(state_in, b, p, d0, a)
                                       : p < end ? load_pack<T, V>(xs + p * a.x_row, valid, a.vec_x) : zero_pack<T, V>();
#pragma unroll
            for (int i = 0; i < V; ++i) { win[j][i] = up(r.v[i]); dp[j][i] = 0; }
        }
        const int last = t1 + H;
        for (int s = t0; s < last; s += 4) {
            Pack<T, V> xr[4], gr[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const bool on = s + k < last && s + k < end;
                xr[k] = on ? load_pack<T, V>(xs + (s + k) * a.x_row, valid, a.vec_x) : zero_pack<T, V>();
                gr[k] = on ? load_pack<T, V>(gs + (s + k) * a.y_row, valid, a.vec_y) : zero_pack<T, V>();
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (s + k >= last) break;
                const bool on = s + k < end;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    win[H][i] = up(xr[k].v[i]);
                    A pre = bias[i];
#pragma unroll
                    for (int j = 0; j < W; ++j) pre += w[i][j] * win[j][i];
                    dp[H][i] = on ? up(gr[k].v[i]) * act_slope(pre, a.silu) : A(0);
                    if (s + k < t1) {
                        db[i] += dp[H][i];
#pragma unroll
                        for (int j = 0; j < W; ++j) dw[i][j] += dp[H][i] * win[j][i];
                    }
                }
                const int t = s + k - H;            /* the row whose gradient is complete now */
                T* to = nullptr;
                if (t >= t0) { if (ds) to = ds + t * a.dx_row; }
                else if (t0 == 0 && dstate_in) to = dstate_in + ((long long)b * H + t + H) * a.channels + d0;
                if (to) {
                    const bool whole = t >= 0 ? a.vec_dx : a.vec_p, add = t >= 0 && acc_dx;
                    const int from_end = t - (end - H);             /* row of the final state that is this row of xp */
                    Pack<T, V> more = zero_pack<T, V>(), have = zero_pack<T, V>(), o;
                    if (dstate_out && from_end >= 0 && from_end < H)
                        more = load_pack<T, V>(dstate_out + ((long long)b * H + from_end) * a.channels + d0, valid, a.vec_p);
                    if (add) have = load_pack<T, V>(to, valid, whole);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        A g = up(more.v[i]);
#pragma unroll
                        for (int j = 0; j < W; ++j) g += w[i][j] * dp[H - j][i];
                        o.v[i] = down<T>(g + up(have.v[i]));
                    }
                    store_pack<T, V>(to, o, valid, whole);
                }
#pragma unroll
                for (int j = 0; j < H; ++j)
#pragma unroll
                    for (int i = 0; i < V; ++i) { win[j][i] = win[j + 1][i]; dp[j][i] = dp[j + 1][i]; }
            }
        }
    }
    if (!parts) return;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        red[ty][W][tx * V + i] = db[i];
#pragma unroll
        for (int j = 0; j < W; ++j) red[ty][j][tx * V + i] = dw[i][j];
    }
    __syncthreads();
    /* part: [channels][W] filter gradients, then [channels] bias gradients */
    A* part = parts + group * (long long)a.channels * (W + 1);
    const int base = d0 - tx * V;
    for (int e = threadIdx.x; e < 32 * V * (W + 1); e += 128) {
        int c, j;
        if (e < 32 * V * W) { c = e / W; j = e - c * W; } else { c = e - 32 * V * W; j = W; }
        if (base + c >= a.channels) continue;
        const A v = ((red[0][j][c] + red[1][j][c]) + red[2][j][c]) + red[3][j][c];
        if (j < W) part[(long long)(base + c) * W + j] = v;
        else part[(long long)a.channels * W + base + c] = v;
    }
}

/* Rows per thread.  A run costs W - 1 (backward: 2 (W - 1)) rows of extra reading, which the longest run makes
 * cheapest; it is halved while the runs do not fill the chip with `warps` warps.  At least 8, so that only the first run of
 * a sequence reaches back to the state. */
int pick_run(long long batch, int len, long long n_vec, int longest, int warps) {
    int run = longest;
    while (run > 8 && batch * ((len + run - 1) / run) * n_vec < (long long)warps * 32) run /= 2;
    return run;
}

template <typename T> int backward_run(const RpbCausalConv* c) {
    const long long n_vec = (c->channels + Width<T>::bwd - 1) / Width<T>::bwd;
    return pick_run(c->batch, c->len, n_vec, 64, SM_COUNT * 16);
}
template <typename T> long long backward_groups(const RpbCausalConv* c) {
    const int run = backward_run<T>(c);
    return ((long long)c->batch * ((c->len + run - 1) / run) + 3) / 4;
}

Rows x_rows(const RpbCausalConv* c, const void* x) { return {x, c->x_batch, c->x_row, c->channels}; }
Rows y_rows(const RpbCausalConv* c, const void* y) { return {y, c->y_batch, c->y_row, c->channels}; }
Rows dx_rows(const RpbCausalConv* c, const void* dx) { return {dx, c->dx_batch, c->dx_row, c->channels}; }
bool packed_ok(const RpbCausalConv* c, const void* p, size_t bytes, size_t es) { return aligned_rows({p, 0, c->channels, c->channels}, 2, 2, es, bytes); }

Args make_args(const RpbCausalConv* c, int v, size_t es, int run) {
    Args a;
    a.batch = c->batch; a.len = c->len; a.channels = c->channels; a.silu = c->activation;
    a.x_batch = c->x_batch; a.x_row = c->x_row; a.y_batch = c->y_batch; a.y_row = c->y_row;
    a.dx_batch = c->dx_batch; a.dx_row = c->dx_row;
    a.run = run; a.runs = (c->len + run - 1) / run;
    a.n_vec = (c->channels + v - 1) / v;
    a.vec_x = a.vec_y = a.vec_dx = a.vec_p = false;
    return a;
}

template <typename T, int W>
int forward_w(void* y, void* state_out, const void* x, const void* w, const void* bias, const void* state_in, const int* lengths,
              const RpbCausalConv* c, cudaStream_t s) {
    constexpr int V = Width<T>::fwd;
    const long long n_vec = (c->channels + V - 1) / V;
    Args a = make_args(c, V, sizeof(T), pick_run(c->batch, c->len, n_vec, 32, SM_COUNT * 16));
    const size_t bytes = sizeof(T) * V;
    a.vec_x = aligned_rows(x_rows(c, x), c->batch, c->len, sizeof(T), bytes);
    a.vec_y = aligned_rows(y_rows(c, y), c->batch, c->len, sizeof(T), bytes);
    a.vec_p = packed_ok(c, state_in, bytes, sizeof(T)) && packed_ok(c, state_out, bytes, sizeof(T));
    const long long items = (long long)c->batch * a.runs * n_vec;
    const int block = items < (long long)SM_COUNT * 128 ? 32 : 128;     /* few items: one warp per block, on more SMs */
    const long long blocks = (items + block - 1) / block;
    if (blocks > 0x7fffffffLL) return refuse("rp_causal_conv_ex", "too many rows for one launch");
    SEQ_CUDA(rpb_launch(forward_kernel<T, W>, dim3((unsigned)blocks), dim3(block), 0, s, 1, reinterpret_cast<T*>(y), reinterpret_cast<T*>(state_out),
                        reinterpret_cast<const T*>(x), reinterpret_cast<const T*>(w), reinterpret_cast<const T*>(bias),
                        reinterpret_cast<const T*>(state_in), lengths, a));
    rpb_count_launches(1);
    return 0;
}

template <typename T, int W>
int backward_w(void* dx, void* dw, void* dbias, void* dstate_in, int accumulate, const void* dy, const void* dstate_out, const void* x,
               const void* w, const void* bias, const void* state_in, const int* lengths, void* ws, const RpbCausalConv* c, cudaStream_t s) {
    typedef typename AccOf<T>::type A;
    constexpr int V = Width<T>::bwd;
    Args a = make_args(c, V, sizeof(T), backward_run<T>(c));
    const size_t bytes = sizeof(T) * V;
    a.vec_x = aligned_rows(x_rows(c, x), c->batch, c->len, sizeof(T), bytes);
    a.vec_y = aligned_rows(y_rows(c, dy), c->batch, c->len, sizeof(T), bytes);
    a.vec_dx = aligned_rows(dx_rows(c, dx), c->batch, c->len, sizeof(T), bytes);
    a.vec_p = packed_ok(c, state_in, bytes, sizeof(T)) && packed_ok(c, dstate_in, bytes, sizeof(T)) && packed_ok(c, dstate_out, bytes, sizeof(T));
    const long long groups = backward_groups<T>(c);
    const int vec_blocks = (a.n_vec + 31) / 32;
    if (groups * vec_blocks > 0x7fffffffLL) return refuse("rp_causal_conv_grad_ex", "too many rows for one launch");
    const bool filter = dw || dbias;
    SEQ_CUDA(rpb_launch(backward_kernel<T, W>, dim3((unsigned)(groups * vec_blocks)), dim3(128), 0, s, 1, reinterpret_cast<T*>(dx),
                        reinterpret_cast<T*>(dstate_in), filter ? reinterpret_cast<A*>(ws) : nullptr, (accumulate & RPB_CONV_ACC_DX) != 0,
                        reinterpret_cast<const T*>(dy), reinterpret_cast<const T*>(dstate_out), reinterpret_cast<const T*>(x),
                        reinterpret_cast<const T*>(w), reinterpret_cast<const T*>(bias), reinterpret_cast<const T*>(state_in), lengths, a, vec_blocks));
    rpb_count_launches(1);
    if (!filter) return 0;
    PartSums d = {};
    d.out[0] = dw; d.first[0] = 0; d.cols[0] = (long long)c->channels * W; d.accumulate[0] = (accumulate & RPB_CONV_ACC_DW) != 0;
    d.out[1] = dbias; d.first[1] = (long long)c->channels * W; d.cols[1] = c->channels; d.accumulate[1] = (accumulate & RPB_CONV_ACC_DBIAS) != 0;
    return sum_parts<T>(d, ws, (int)groups, (long long)c->channels * (W + 1), s);
}

template <typename T, typename F> int by_width(int width, F f) {
    switch (width) {
        case 1: return f(std::integral_constant<int, 1>());
        case 2: return f(std::integral_constant<int, 2>());
        case 3: return f(std::integral_constant<int, 3>());
        case 4: return f(std::integral_constant<int, 4>());
        case 5: return f(std::integral_constant<int, 5>());
        case 6: return f(std::integral_constant<int, 6>());
        case 7: return f(std::integral_constant<int, 7>());
        case 8: return f(std::integral_constant<int, 8>());
    }
    return -1;
}

const char* bad_geometry(const RpbCausalConv* c, DType dtype) {
    if (!c) return "no geometry";
    if (!rpb_dtype_size((int)dtype)) return "unknown element type";
    if (c->batch <= 0 || c->len <= 0 || c->channels <= 0) return "batch, len and channels must be positive";
    if (c->width < 1 || c->width > 8) return "width must be 1 to 8";
    if (c->activation != 0 && c->activation != 1) return "activation must be 0 (none) or 1 (SiLU)";
    return nullptr;
}

template <typename T> long long ws_bytes(const RpbCausalConv* c) {
    return backward_groups<T>(c) * c->channels * (c->width + 1) * (long long)sizeof(typename AccOf<T>::type);
}

}  // namespace rpb_conv1d

using namespace rpb_seq;
using namespace rpb_conv1d;

extern "C" {

void rpb_causal_conv_packed(RpbCausalConv* c, int batch, int len, int channels, int width, int activation) {
    memset(c, 0, sizeof(*c));
    c->batch = batch; c->len = len; c->channels = channels; c->width = width; c->activation = activation;
    c->x_row = c->y_row = c->dx_row = channels;
    c->x_batch = c->y_batch = c->dx_batch = (long long)len * channels;
}

int rp_causal_conv_ex(void* y, void* state_out, const void* x, const void* w, const void* bias, const void* state_in, const int* lengths,
                      const RpbCausalConv* c, DType dtype, int device_id, void* stream) {
    const char* name = "rp_causal_conv_ex";
    const char* why = bad_geometry(c, dtype);
    if (why) return refuse(name, why);
    if (!y || !x || !w) return refuse(name, "y, x and w are needed");
    if (device_id < 0) return refuse(name, "needs a CUDA device (no CPU path in this library)");
    const Rows rx = x_rows(c, x), ry = y_rows(c, y);
    if (!readable(rx, c->batch, c->len)) return refuse(name, "strides of x");
    if (!writable(ry, c->batch, c->len)) return refuse(name, "strides of y");
    if (overlaps(ry, rx, c->batch, c->len, rpb_dtype_size((int)dtype))) return refuse(name, "y overlaps x");
    DeviceScope scope;
    if (scope.enter(device_id)) return refuse(name, "no such device");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    switch ((int)dtype) {
#define CASE(code, T) case code: return by_width<T>(c->width, [&](auto W) { return forward_w<T, decltype(W)::value>(y, state_out, x, w, bias, state_in, lengths, c, s); });
        CASE(DTYPE_FLOAT32, float) CASE(DTYPE_FLOAT64, double) CASE(DTYPE_FLOAT16, __half) CASE(DTYPE_BFLOAT16, __nv_bfloat16)
#undef CASE
    }
    return -1;
}

long long rp_causal_conv_ws_bytes(const RpbCausalConv* c, DType dtype) {
    const char* why = bad_geometry(c, dtype);
    if (why) return refuse("rp_causal_conv_ws_bytes", why);
    switch ((int)dtype) {
        case DTYPE_FLOAT32: return ws_bytes<float>(c);
        case DTYPE_FLOAT64: return ws_bytes<double>(c);
        default: return ws_bytes<__nv_bfloat16>(c);
    }
}

int rp_causal_conv_grad_ex(void* dx, void* dw, void* dbias, void* dstate_in, int accumulate, const void* dy, const void* dstate_out,
                           const void* x, const void* w, const void* bias, const void* state_in, const int* lengths, void* ws,
                           const RpbCausalConv* c, DType dtype, int device_id, void* stream) {
    const char* name = "rp_causal_conv_grad_ex";
    const char* why = bad_geometry(c, dtype);
    if (why) return refuse(name, why);
    if (!dy || !x || !w) return refuse(name, "dy, x and w are needed");
    if (!dx && !dw && !dbias && !dstate_in) return refuse(name, "no gradient is wanted");
    if ((dw || dbias) && !ws) return refuse(name, "the filter's gradients need a workspace");
    if (device_id < 0) return refuse(name, "needs a CUDA device (no CPU path in this library)");
    const Rows rx = x_rows(c, x), rg = y_rows(c, dy), rd = dx_rows(c, dx);
    const size_t es = rpb_dtype_size((int)dtype);
    if (!readable(rx, c->batch, c->len)) return refuse(name, "strides of x");
    if (!readable(rg, c->batch, c->len)) return refuse(name, "strides of dy");
    if (dx && !writable(rd, c->batch, c->len)) return refuse(name, "strides of dx");
    if (overlaps(rd, rx, c->batch, c->len, es) || overlaps(rd, rg, c->batch, c->len, es)) return refuse(name, "dx overlaps x or dy");
    if (dstate_in && (dstate_in == dstate_out || dstate_in == state_in)) return refuse(name, "dstate_in overlaps dstate_out or state_in");
    DeviceScope scope;
    if (scope.enter(device_id)) return refuse(name, "no such device");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    switch ((int)dtype) {
#define CASE(code, T) case code: return by_width<T>(c->width, [&](auto W) { return backward_w<T, decltype(W)::value>(dx, dw, dbias, dstate_in, accumulate, dy, dstate_out, x, w, bias, state_in, lengths, ws, c, s); });
        CASE(DTYPE_FLOAT32, float) CASE(DTYPE_FLOAT64, double) CASE(DTYPE_FLOAT16, __half) CASE(DTYPE_BFLOAT16, __nv_bfloat16)
#undef CASE
    }
    return -1;
}

}  // extern "C"
