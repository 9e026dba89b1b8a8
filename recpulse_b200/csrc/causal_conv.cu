/*
 * Short causal convolution along a sequence, one filter per channel, with its SiLU and its gradients:
 *   pre[b,t,d] = bias[d] + sum over j < width of w[d,j] * xp[b,t+j,d],   y = pre or pre / (1 + exp(-pre))
 * where xp is x behind width-1 earlier rows (the state of the sequence, or zeros).  Its floor is memory: 41 us for reading and writing
 * 4 x 4096 x 4096 bf16 at the measured copy rate (about 30 with the lengths measured); the forward kernel takes 71 us there (16 bytes
 * per thread and window moves took 119 us).  About 25 instructions per value are some 32 us of issue; five warps per scheduler at 95
 * registers do not overlap them with the loads that they wait for (issue slots 48% busy).
 */
#include "seq_common.cuh"

namespace rpb_conv1d {

using namespace rpb_seq;

struct Args {
    int batch, len, channels, silu, width;
    long long x_batch, x_row, y_batch, y_row, dx_batch, dx_row;
    int run, runs;          /* rows per thread, and such runs per sequence */
    int vec_blocks;         /* warps that cover the channels */
};

/* Channels of a thread: 8 bytes of a 16-bit row (16 bytes needed twice the registers and ran at half the warps), 16 of others. */
template <typename T> struct Width { static constexpr int v = sizeof(T) == 2 ? 4 : 16 / sizeof(T); };

__device__ __forceinline__ int row_end(const int* lengths, int b, int len) {
    if (!lengths) return len;
    const int n = lengths[b];
    return n < 0 ? 0 : n > len ? len : n;
}

template <typename A> __device__ __forceinline__ A act_slope(A pre, int silu) {
    if (!silu) return A(1);
    const A s = logistic(pre);
    return s * (A(1) + pre * (A(1) - s));
}

/* A thread's V channels.  VEC: neighbours, moved as one pack (every row aligned, V divides the channels); else every 32nd one, so
 * that a warp's single values are neighbours. */
template <typename T, bool VEC> struct Lane {
    static constexpr int V = Width<T>::v;
    int d0, channels;
    __device__ __forceinline__ int channel(int i) const { return VEC ? d0 + i : d0 + 32 * i; }
    __device__ __forceinline__ bool has(int i) const { return VEC ? d0 < channels : channel(i) < channels; }
    /* `row`: the row's first channel */
    __device__ __forceinline__ Pack<T, V> load(const T* row, bool on) const {
        Pack<T, V> p = zero_pack<T, V>();
        if (VEC) {
            if (on && has(0)) p = *reinterpret_cast<const Pack<T, V>*>(row + d0);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (on && has(i)) p.v[i] = row[channel(i)];
        }
        return p;
    }
    __device__ __forceinline__ void store(T* row, const Pack<T, V>& p) const {
        if (VEC) {
            if (has(0)) *reinterpret_cast<Pack<T, V>*>(row + d0) = p;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (has(i)) row[channel(i)] = p.v[i];
        }
    }
};

/* Where a thread works: one warp per run of rows, four runs per block. */
template <typename T, bool VEC> struct Place {
    Lane<T, VEC> lane;
    long long group, seq;
    int b, t0, t1;
    bool on;
    __device__ __forceinline__ explicit Place(const Args& a) {
        const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, first = (int)(blockIdx.x % a.vec_blocks) * 32 * Width<T>::v;
        lane.channels = a.channels;
        lane.d0 = VEC ? first + tx * Width<T>::v : first + tx;
        group = blockIdx.x / a.vec_blocks;
        seq = group * (blockDim.x >> 5) + ty;
        on = seq < (long long)a.batch * a.runs;
        b = on ? (int)(seq / a.runs) : 0;
        t0 = on ? (int)(seq - (long long)b * a.runs) * a.run : 0;
        t1 = t0 + a.run < a.len ? t0 + a.run : a.len;
    }
};

/* The filter of up to W taps, behind W - width zeros that no product is formed with (`skip`), and the bias. */
template <typename T, int W, bool VEC, typename A>
__device__ __forceinline__ void load_taps(A (&w)[W][Width<T>::v], A (&bias)[Width<T>::v], const T* wt, const T* bt, const Lane<T, VEC>& lane, int width) {
#pragma unroll
    for (int i = 0; i < Width<T>::v; ++i) {
        const bool on = lane.has(i);
        const long long c = lane.channel(i);
#pragma unroll
        for (int j = 0; j < W; ++j) w[j][i] = on && j >= W - width ? up(wt[c * width + j - (W - width)]) : A(0);
        bias[i] = on && bt ? up(bt[c]) : A(0);
    }
}

/* Row p of xp: of x within the sequence, in front of it of the sequence's state (row p + width - 1), else zeros. */
template <typename T, bool VEC>
__device__ __forceinline__ Pack<T, Width<T>::v> row_of(const T* x, const T* state, int p, int end, const Lane<T, VEC>& lane, const Args& a) {
    const int s = p + a.width - 1;
    if (p >= 0) return lane.load(x + p * a.x_row, p < end);
    return lane.load(state + (long long)s * a.channels, state && s >= 0);
}

/* Rows at a time, the next ones' values on their way meanwhile: 4 forward (2: 79 us instead of 71 at 4 x 4096 x 4096 bf16, 8: 103),
 * 2 backward.  Forward and backward kernels together, replayed from a graph, with 2 and with 4 rows backward: 47 and 64 us at
 * 3 x 1999 x 1531 x 3 taps f16 (rows off the boundaries), 138 and 130 at 2 x 2048 x 4096 x 4 taps bf16, 73 and 72 at 2 x 2048 x
 * 1024 x 8 taps float32. */
constexpr int FORWARD_ROWS = 4, BACKWARD_ROWS = 2;

/* The last W - 1 rows of x are kept in registers, so that x is read once but for W - 1 rows in front of each run. */
template <typename T, int W, bool VEC>
__global__ void __launch_bounds__(128) forward_kernel(T* __restrict__ y, T* state_out, const T* __restrict__ x, const T* __restrict__ wt,
                                                      const T* __restrict__ bt, const T* state_in, const int* __restrict__ lengths, Args a) {
    typedef typename AccOf<T>::type A;
    constexpr int V = Width<T>::v, H = W - 1, U = FORWARD_ROWS;
    rpb_pdl_trigger();
    rpb_pdl_wait();
    const Place<T, VEC> pl(a);
    if (!pl.on) return;
    const Lane<T, VEC>& lane = pl.lane;
    const int end = row_end(lengths, pl.b, a.len), skip = W - a.width, keep = a.width - 1;
    const T* xs = x + pl.b * a.x_batch;
    T* ys = y + pl.b * a.y_batch;
    const T* first = state_in ? state_in + (long long)pl.b * keep * a.channels : nullptr;
    int t = pl.t0;
    const int stop = pl.t1 < end ? pl.t1 : end;
    if (t < end) {
        const T* xn = xs + (t + U) * a.x_row;
        T* yt = ys + t * a.y_row;
        A w[W][V], bias[V], win[H + U][V];          /* win[j]: row t - H + j */
        load_taps<T, W, VEC>(w, bias, wt, bt, lane, a.width);
        Pack<T, V> next[U], early[H];
#pragma unroll
        for (int j = 0; j < H; ++j) early[j] = j >= skip ? row_of(xs, first, t - H + j, end, lane, a) : zero_pack<T, V>();
#pragma unroll
        for (int k = 0; k < U; ++k) next[k] = lane.load(xs + (t + k) * a.x_row, t + k < stop);
#pragma unroll
        for (int j = 0; j < H; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) win[j][i] = up(early[j].v[i]);
        for (; t < stop; t += U) {
#pragma unroll
            for (int k = 0; k < U; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) win[H + k][i] = up(next[k].v[i]);
#pragma unroll
            for (int k = 0; k < U; ++k) next[k] = lane.load(xn + k * a.x_row, t + U + k < stop);
            xn += U * a.x_row;
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (t + k >= stop) break;
                A o[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    A pre = bias[i];
#pragma unroll
                    for (int j = 0; j < W; ++j)
                        if (j >= skip) pre += w[j][i] * win[k + j][i];
                    o[i] = pre;
                }
                if (a.silu) {
#pragma unroll
                    for (int i = 0; i < V; ++i) o[i] *= logistic(o[i]);
                }
                lane.store(yt + k * a.y_row, store_form<T, V>(o));
            }
            yt += U * a.y_row;
#pragma unroll
            for (int j = 0; j < H; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) win[j][i] = win[j + U][i];
        }
    }
    for (t = pl.t0 > end ? pl.t0 : end; t < pl.t1; ++t) lane.store(ys + t * a.y_row, zero_pack<T, V>());
    if (state_out && pl.t0 == 0) {
        /* the last rows of xp, by the only run that reads the old state; all read before the first is written: state_out may be
         * state_in */
        Pack<T, V> last[H];
#pragma unroll
        for (int j = 0; j < H; ++j) last[j] = j < keep ? row_of(xs, first, end - keep + j, end, lane, a) : zero_pack<T, V>();
#pragma unroll
        for (int j = 0; j < H; ++j)
            if (j < keep) lane.store(state_out + ((long long)pl.b * keep + j) * a.channels, last[j]);
    }
}

/* With dpre = dy act'(pre), 0 outside the sequence:
 *   dxp[p] = sum over j of w[j] dpre[p - j],   dw[j] = sum over t of dpre[t] xp[t + j],   dbias = sum of dpre.
 * A thread walks its rows upwards and W - 1 rows further, computes dpre of each row again from x and emits the gradient
 * of the row W - 1 behind; the run that begins a sequence emits the state's gradient in the same way.  The filter's
 * gradients of a block's four runs are added in shared memory and written as one part; sum_parts adds the parts. */
template <typename T, int W, bool VEC>
__global__ void __launch_bounds__(128) backward_kernel(T* dx, T* dstate_in, typename AccOf<T>::type* __restrict__ parts, int acc_dx,
                                                       const T* __restrict__ dy, const T* __restrict__ dstate_out, const T* __restrict__ x,
                                                       const T* __restrict__ wt, const T* __restrict__ bt, const T* __restrict__ state_in,
                                                       const int* __restrict__ lengths, Args a) {
    typedef typename AccOf<T>::type A;
    constexpr int V = Width<T>::v, H = W - 1, U = BACKWARD_ROWS;
    __shared__ A red[4][W + 1][32 * V + 1];
    rpb_pdl_trigger();
    rpb_pdl_wait();
    const Place<T, VEC> pl(a);
    const Lane<T, VEC>& lane = pl.lane;
    const int skip = W - a.width, keep = a.width - 1;
    A dw[W][V], db[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        db[i] = 0;
#pragma unroll
        for (int j = 0; j < W; ++j) dw[j][i] = 0;
    }
    if (pl.on) {
        const int end = row_end(lengths, pl.b, a.len);
        const T* xs = x + pl.b * a.x_batch;
        const T* gs = dy + pl.b * a.y_batch;
        T* ds = dx ? dx + pl.b * a.dx_batch : nullptr;
        const T* first = state_in ? state_in + (long long)pl.b * keep * a.channels : nullptr;
        const T* more_from = dstate_out ? dstate_out + (long long)pl.b * keep * a.channels : nullptr;
        T* to_state = dstate_in ? dstate_in + (long long)pl.b * keep * a.channels : nullptr;
        A w[W][V], bias[V], win[H + U][V], dp[H + U][V];        /* row t - H + j; dp: of dpre */
        load_taps<T, W, VEC>(w, bias, wt, bt, lane, a.width);
        Pack<T, V> xn[U], gn[U], early[H];
        int t = pl.t0;
        const int stop = pl.t1 + H;
        auto fetch = [&](int s) {
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const bool on = s + k < stop && s + k < end;
                xn[k] = lane.load(xs + (s + k) * a.x_row, on);
                gn[k] = lane.load(gs + (s + k) * a.y_row, on);
            }
        };
#pragma unroll
        for (int j = 0; j < H; ++j) early[j] = j >= skip ? row_of(xs, first, t - H + j, end, lane, a) : zero_pack<T, V>();
        fetch(t);
#pragma unroll
        for (int j = 0; j < H; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) { win[j][i] = up(early[j].v[i]); dp[j][i] = 0; }
        /* U rows from t on.  INNER: all of them are the run's own, and every product of their gradients is with a row of the sequence;
         * else each is looked at, since 0 times an infinity of x or of the filter is to be formed nowhere. */
        auto rows = [&](auto inner, const Pack<T, V> (&g)[U]) {
            constexpr bool INNER = decltype(inner)::value;
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int s = t + k;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    A pre = bias[i];
#pragma unroll
                    for (int j = 0; j < W; ++j)
                        if (j >= skip) pre += w[j][i] * win[k + j][i];
                    const A d = INNER || (s < stop && s < end) ? up(g[k].v[i]) * act_slope(pre, a.silu) : A(0);
                    dp[H + k][i] = d;
                    if (INNER || (s < pl.t1 && s < end)) {
                        db[i] += d;
#pragma unroll
                        for (int j = 0; j < W; ++j)
                            if (j >= skip) dw[j][i] += d * win[k + j][i];
                    }
                }
                const int r = s - H;                /* the row whose gradient is complete now */
                T* to = nullptr;
                if (!INNER && r >= pl.t1) break;
                if (r >= pl.t0) { if (ds) to = ds + r * a.dx_row; }
                else if (!INNER && pl.t0 == 0 && to_state && r >= -keep) to = to_state + (long long)(r + keep) * a.channels;
                if (!to) continue;
                A v[V];
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = 0;
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    if (j < skip || !(INNER || (s - j >= 0 && s - j < end))) continue;
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] += w[j][i] * dp[H + k - j][i];
                }
                const int from_end = r - (end - keep);              /* row of the final state that is this row of xp */
                if (!INNER && more_from && from_end >= 0 && from_end < keep) {
                    const Pack<T, V> more = lane.load(more_from + (long long)from_end * a.channels, true);
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] += up(more.v[i]);
                }
                if (r >= 0 && acc_dx) {
                    const Pack<T, V> have = lane.load(to, true);
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] += up(have.v[i]);
                }
                lane.store(to, store_form<T, V>(v));
            }
        };
        for (; t < stop; t += U) {
            Pack<T, V> g[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                g[k] = gn[k];
#pragma unroll
                for (int i = 0; i < V; ++i) win[H + k][i] = up(xn[k].v[i]);
            }
            fetch(t + U);
            if (t >= H && t + U <= pl.t1 && t + U <= end) rows(std::true_type(), g);
            else rows(std::false_type(), g);
#pragma unroll
            for (int j = 0; j < H; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) { win[j][i] = win[j + U][i]; dp[j][i] = dp[j + U][i]; }
        }
    }
    if (!parts) return;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = VEC ? tx * V + i : tx + 32 * i;
        red[ty][W][c] = db[i];
#pragma unroll
        for (int j = 0; j < W; ++j) red[ty][j][c] = dw[j][i];
    }
    __syncthreads();
    /* part: [channels][width] filter gradients, then [channels] bias gradients */
    A* part = parts + pl.group * (long long)a.channels * (a.width + 1);
    const int base = (int)(blockIdx.x % a.vec_blocks) * 32 * V;
    for (int e = threadIdx.x; e < 32 * V * (a.width + 1); e += 128) {
        int c, j;
        if (e < 32 * V * a.width) { c = e / a.width; j = e - c * a.width; } else { c = e - 32 * V * a.width; j = a.width; }
        if (base + c >= a.channels) continue;
        const int from = j < a.width ? j + skip : W;
        const A v = ((red[0][from][c] + red[1][from][c]) + red[2][from][c]) + red[3][from][c];
        if (j < a.width) part[(long long)(base + c) * a.width + j] = v;
        else part[(long long)a.channels * a.width + base + c] = v;
    }
}

/* Rows per thread.  A run costs W - 1 (backward: 2 (W - 1)) rows of extra reading, which the longest run makes
 * cheapest; it is halved while the runs do not fill the chip with `warps` warps: 16 per SM forward, 8 backward, whose runs cost
 * twice as much (with 8 and with 16, at the three shapes above: 47 and 51, 138 and 124, 73 and 98 us).  At least 8, so that only
 * the first run of a sequence reaches back to the state. */
int pick_run(long long batch, int len, long long n_vec, int longest, int warps) {
    int run = longest;
    while (run > 8 && batch * ((len + run - 1) / run) * n_vec < (long long)warps * 32) run /= 2;
    return run;
}

template <typename T> int backward_run(const RpbCausalConv* c) {
    return pick_run(c->batch, c->len, (c->channels + Width<T>::v - 1) / Width<T>::v, 64, SM_COUNT * 8);
}
template <typename T> long long backward_groups(const RpbCausalConv* c) {
    const int run = backward_run<T>(c);
    return ((long long)c->batch * ((c->len + run - 1) / run) + 3) / 4;
}

Rows x_rows(const RpbCausalConv* c, const void* x) { return {x, c->x_batch, c->x_row, c->channels}; }
Rows y_rows(const RpbCausalConv* c, const void* y) { return {y, c->y_batch, c->y_row, c->channels}; }
Rows dx_rows(const RpbCausalConv* c, const void* dx) { return {dx, c->dx_batch, c->dx_row, c->channels}; }

long long state_elems(const RpbCausalConv* c) { return (long long)c->batch * (c->width - 1) * c->channels; }

/* Whether every row of an operand (a packed state: p, 0 strides) can be moved in packs. */
template <typename T> bool packs_ok(const RpbCausalConv* c, const Rows& r) {
    return !r.p || aligned_rows(r, c->batch, c->len, sizeof(T), sizeof(T) * Width<T>::v);
}
template <typename T> bool state_ok(const RpbCausalConv* c, const void* p) {
    return !p || reinterpret_cast<uintptr_t>(p) % (sizeof(T) * Width<T>::v) == 0;
}

template <typename T> Args make_args(const RpbCausalConv* c, int run) {
    Args a;
    a.batch = c->batch; a.len = c->len; a.channels = c->channels; a.silu = c->activation; a.width = c->width;
    a.x_batch = c->x_batch; a.x_row = c->x_row; a.y_batch = c->y_batch; a.y_row = c->y_row;
    a.dx_batch = c->dx_batch; a.dx_row = c->dx_row;
    a.run = run; a.runs = (c->len + run - 1) / run;
    a.vec_blocks = (c->channels + 32 * Width<T>::v - 1) / (32 * Width<T>::v);
    return a;
}

template <typename T, int W, bool VEC>
int forward_w(void* y, void* state_out, const void* x, const void* w, const void* bias, const void* state_in, const int* lengths,
              const RpbCausalConv* c, cudaStream_t s) {
    const Args a = make_args<T>(c, pick_run(c->batch, c->len, (c->channels + Width<T>::v - 1) / Width<T>::v, 64, SM_COUNT * 16));
    const long long warps = (long long)c->batch * a.runs * a.vec_blocks;
    const int per = warps < SM_COUNT * 4 ? 1 : 4;                  /* few warps: one per block, on more SMs */
    const long long blocks = ((long long)c->batch * a.runs + per - 1) / per * a.vec_blocks;
    if (blocks > 0x7fffffffLL) return refuse("rp_causal_conv_ex", "too many rows for one launch");
    SEQ_CUDA(rpb_launch(forward_kernel<T, W, VEC>, dim3((unsigned)blocks), dim3(32 * per), 0, s, 1, reinterpret_cast<T*>(y), reinterpret_cast<T*>(state_out),
                        reinterpret_cast<const T*>(x), reinterpret_cast<const T*>(w), reinterpret_cast<const T*>(bias),
                        reinterpret_cast<const T*>(state_in), lengths, a));
    rpb_count_launches(1);
    return 0;
}

template <typename T, int W, bool VEC>
int backward_w(void* dx, void* dw, void* dbias, void* dstate_in, int accumulate, const void* dy, const void* dstate_out, const void* x,
               const void* w, const void* bias, const void* state_in, const int* lengths, void* ws, const RpbCausalConv* c, cudaStream_t s) {
    typedef typename AccOf<T>::type A;
    const Args a = make_args<T>(c, backward_run<T>(c));
    const long long groups = backward_groups<T>(c);
    if (groups * a.vec_blocks > 0x7fffffffLL) return refuse("rp_causal_conv_grad_ex", "too many rows for one launch");
    const bool filter = dw || dbias;
    SEQ_CUDA(rpb_launch(backward_kernel<T, W, VEC>, dim3((unsigned)(groups * a.vec_blocks)), dim3(128), 0, s, 1, reinterpret_cast<T*>(dx),
                        reinterpret_cast<T*>(dstate_in), filter ? reinterpret_cast<A*>(ws) : nullptr, (accumulate & RPB_CONV_ACC_DX) != 0,
                        reinterpret_cast<const T*>(dy), reinterpret_cast<const T*>(dstate_out), reinterpret_cast<const T*>(x),
                        reinterpret_cast<const T*>(w), reinterpret_cast<const T*>(bias), reinterpret_cast<const T*>(state_in), lengths, a));
    rpb_count_launches(1);
    if (!filter) return 0;
    const long long D = c->channels;
    PartSums d = {};
    d.out[0] = dw; d.first[0] = 0; d.cols[0] = D * c->width; d.accumulate[0] = (accumulate & RPB_CONV_ACC_DW) != 0;
    d.out[1] = dbias; d.first[1] = D * c->width; d.cols[1] = D; d.accumulate[1] = (accumulate & RPB_CONV_ACC_DBIAS) != 0;
    return sum_parts<T>(d, ws, (int)groups, D * (c->width + 1), s);
}

/* The kernels are built for 2, 3, 4 and 8 taps; fewer are the last ones of these. */
template <typename T, typename F> int by_width(int width, bool vec, F f) {
#define CASE(n) if (width <= n) return vec ? f(std::integral_constant<int, n>(), std::true_type()) : f(std::integral_constant<int, n>(), std::false_type());
    CASE(2) CASE(3) CASE(4) CASE(8)
#undef CASE
    return -1;
}

template <typename T>
int run_forward(void* y, void* state_out, const void* x, const void* w, const void* bias, const void* state_in, const int* lengths,
                const RpbCausalConv* c, cudaStream_t s) {
    const bool vec = c->channels % Width<T>::v == 0 && packs_ok<T>(c, x_rows(c, x)) && packs_ok<T>(c, y_rows(c, y)) && state_ok<T>(c, state_in) &&
                     state_ok<T>(c, state_out);
    return by_width<T>(c->width, vec, [&](auto n, auto p) {
        return forward_w<T, decltype(n)::value, decltype(p)::value>(y, state_out, x, w, bias, state_in, lengths, c, s);
    });
}
template <typename T>
int run_backward(void* dx, void* dw, void* dbias, void* dstate_in, int accumulate, const void* dy, const void* dstate_out, const void* x,
                 const void* w, const void* bias, const void* state_in, const int* lengths, void* ws, const RpbCausalConv* c, cudaStream_t s) {
    const bool vec = c->channels % Width<T>::v == 0 && packs_ok<T>(c, x_rows(c, x)) && packs_ok<T>(c, y_rows(c, dy)) && packs_ok<T>(c, dx_rows(c, dx)) &&
                     state_ok<T>(c, state_in) && state_ok<T>(c, dstate_in) && state_ok<T>(c, dstate_out);
    return by_width<T>(c->width, vec, [&](auto n, auto p) {
        return backward_w<T, decltype(n)::value, decltype(p)::value>(dx, dw, dbias, dstate_in, accumulate, dy, dstate_out, x, w, bias, state_in, lengths,
                                                                     ws, c, s);
    });
}

const char* bad_geometry(const RpbCausalConv* c, DType dtype) {
    if (!c) return "no geometry";
    if (!rpb_dtype_size((int)dtype)) return "unknown element type";
    if (c->batch <= 0 || c->len <= 0 || c->channels <= 0) return "batch, len and channels must be positive";
    if (c->batch > 1 << 30 || c->len > 1 << 30 || c->channels > 1 << 24) return "batch or len above 2^30, or channels above 2^24";
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
    const size_t es = rpb_dtype_size((int)dtype);
    const long long kept = state_elems(c);
    const Area outs[] = {strided("y", ry, c->batch, c->len, es), packed("state_out", state_out, kept, es, state_in)};
    const Area ins[] = {strided("x", rx, c->batch, c->len, es), packed("w", w, (long long)c->channels * c->width, es), packed("bias", bias, c->channels, es),
                        packed("state_in", state_in, kept, es), packed("lengths", lengths, c->batch, sizeof(int))};
    if (refuse_buffers(name, outs, ins)) return -1;
    DeviceScope scope;
    if (scope.enter(device_id)) return refuse(name, "no such device");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    switch ((int)dtype) {
#define CASE(code, T) case code: return run_forward<T>(y, state_out, x, w, bias, state_in, lengths, c, s);
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
    const size_t es = rpb_dtype_size((int)dtype), as = dtype == DTYPE_FLOAT64 ? 8 : 4;
    if (!readable(rx, c->batch, c->len)) return refuse(name, "strides of x");
    if (!readable(rg, c->batch, c->len)) return refuse(name, "strides of dy");
    if (dx && !writable(rd, c->batch, c->len)) return refuse(name, "strides of dx");
    const long long kept = state_elems(c), taps = (long long)c->channels * c->width;
    const bool filter = dw || dbias;
    const Area outs[] = {strided("dx", rd, c->batch, c->len, es), packed("dw", dw, taps, es), packed("dbias", dbias, c->channels, es),
                         packed("dstate_in", dstate_in, kept, es), packed("ws", filter ? ws : nullptr, filter ? rp_causal_conv_ws_bytes(c, dtype) / (long long)as : 0, as)};
    const Area ins[] = {strided("dy", rg, c->batch, c->len, es), strided("x", rx, c->batch, c->len, es), packed("w", w, taps, es),
                        packed("bias", bias, c->channels, es), packed("state_in", state_in, kept, es), packed("dstate_out", dstate_out, kept, es),
                        packed("lengths", lengths, c->batch, sizeof(int))};
    if (refuse_buffers(name, outs, ins)) return -1;
    DeviceScope scope;
    if (scope.enter(device_id)) return refuse(name, "no such device");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    switch ((int)dtype) {
#define CASE(code, T) case code: return run_backward<T>(dx, dw, dbias, dstate_in, accumulate, dy, dstate_out, x, w, bias, state_in, lengths, ws, c, s);
        CASE(DTYPE_FLOAT32, float) CASE(DTYPE_FLOAT64, double) CASE(DTYPE_FLOAT16, __half) CASE(DTYPE_BFLOAT16, __nv_bfloat16)
#undef CASE
    }
    return -1;
}

}  // extern "C"
