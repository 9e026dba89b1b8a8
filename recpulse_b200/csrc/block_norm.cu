/*
 * The norms around a block, with its gate and the scaled add to the residual, one pass over each row:
 *   v = u z / (1 + exp(-z)) (or u),  s = v rsqrt(mean v^2 + eps_after) w_after (or v),  out = r + scale s,
 *   y = out rsqrt(mean out^2 + eps_before) w_before.
 * Backward: with t = v i (i = rsqrt(mean v^2 + eps)) and m the gradient of t, dv = i (m - t mean(m t)); y's norm likewise.
 * A block of threads holds a whole row in registers, so each operand is read once and the row's sums are taken from there.
 */
#include "seq_common.cuh"

namespace rpb_norm {

using namespace rpb_seq;

constexpr int MAX_CHANNELS = 16384;

struct Args {
    long long rows;
    int channels;
    double eps_after, eps_before;
    long long u_row, z_row, r_row, out_row, y_row, du_row, dz_row, dr_row;
    bool vec;               /* every operand can be moved in whole packs */
};

template <typename T> struct Width { static constexpr int v = 16 / sizeof(T); };

__device__ __forceinline__ float rsqrt_of(float v) { return rsqrtf(v); }
__device__ __forceinline__ double rsqrt_of(double v) { return rsqrt(v); }

/* Sum over the block; every thread gets it.  The two halves of the buffer take turns, so that one barrier per
 * sum is enough: a half is written again only behind the next sum's barrier. */
template <typename A> __device__ __forceinline__ A block_sum(A v, A (*buffer)[32], int& turn) {
#pragma unroll
    for (int m = 16; m >= 1; m /= 2) v += __shfl_xor_sync(0xffffffffu, v, m);
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    A* slots = buffer[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    A s = (threadIdx.x & 31) < warps ? slots[threadIdx.x & 31] : A(0);
#pragma unroll
    for (int m = 16; m >= 1; m /= 2) s += __shfl_xor_sync(0xffffffffu, s, m);
    return s;
}

/* pack k of a thread: channels (k * blockDim + thread) * V .. */
template <int V> __device__ __forceinline__ int channel_of(int k) { return (k * blockDim.x + threadIdx.x) * V; }

template <typename T, int NV, typename A = typename AccOf<T>::type>
__device__ __forceinline__ void load_row(Pack<T, Width<T>::v> (&p)[NV], const T* row, const Args& a) {
    constexpr int V = Width<T>::v;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = channel_of<V>(k);
        p[k] = row ? load_pack<T, V>(row + c, a.channels - c, a.vec) : zero_pack<T, V>();
    }
}

template <typename T, int NV>
__global__ void __launch_bounds__(512) forward_kernel(T* __restrict__ out, T* __restrict__ y, const T* __restrict__ u, const T* __restrict__ z, const T* __restrict__ w_after,
                               const T* __restrict__ scale, const T* __restrict__ r, const T* __restrict__ w_before, Args a) {
    typedef typename AccOf<T>::type A;
    constexpr int V = Width<T>::v;
    __shared__ A buffer[2][32];
    int turn = 0;
    rpb_pdl_trigger();
    rpb_pdl_wait();
    const A inv = A(1) / A(a.channels);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        Pack<T, V> up_[NV], zp[NV], rp[NV];
        load_row<T, NV>(up_, u + row * a.u_row, a);
        load_row<T, NV>(zp, z ? z + row * a.z_row : nullptr, a);
        load_row<T, NV>(rp, r ? r + row * a.r_row : nullptr, a);
        A v[NV][V], sq = 0;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[k][i] = up(up_[k].v[i]);
                if (z) { const A g = up(zp[k].v[i]); v[k][i] *= g * logistic(g); }
                sq += v[k][i] * v[k][i];
            }
        const A i1 = w_after ? rsqrt_of(block_sum(sq, buffer, turn) * inv + A(a.eps_after)) : A(1);
        sq = 0;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = channel_of<V>(k), valid = a.channels - c;
            const Pack<T, V> wp = w_after ? load_pack<T, V>(w_after + c, valid, a.vec) : zero_pack<T, V>();
            const Pack<T, V> sp = scale ? load_pack<T, V>(scale + c, valid, a.vec) : zero_pack<T, V>();
            Pack<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                A s = v[k][i];
                if (w_after) s = s * i1 * up(wp.v[i]);
                if (scale) s *= up(sp.v[i]);
                v[k][i] = i < valid ? up(rp[k].v[i]) + s : A(0);
                o.v[i] = down<T>(v[k][i]);
                sq += v[k][i] * v[k][i];
            }
            if (out) store_pack<T, V>(out + row * a.out_row + c, o, valid, a.vec);
        }
        if (!y) continue;
        const A i2 = rsqrt_of(block_sum(sq, buffer, turn) * inv + A(a.eps_before));
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = channel_of<V>(k), valid = a.channels - c;
            const Pack<T, V> wp = load_pack<T, V>(w_before + c, valid, a.vec);
            Pack<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] = down<T>(v[k][i] * i2 * up(wp.v[i]));
            store_pack<T, V>(y + row * a.y_row + c, o, valid, a.vec);
        }
    }
}

/* Each block takes every gridDim-th row and keeps its part of the weights' gradients in registers; sum_parts adds the
 * blocks' parts [3][channels]: w_after, scale, w_before. */
template <typename T, int NV>
__global__ void __launch_bounds__(512) backward_kernel(T* du, T* dz, T* dr, typename AccOf<T>::type* __restrict__ parts, int acc_du, int acc_dz, int acc_dr,
                                const T* __restrict__ dout, const T* __restrict__ dy, const T* __restrict__ u, const T* __restrict__ z,
                                const T* __restrict__ w_after, const T* __restrict__ scale, const T* __restrict__ r, const T* __restrict__ w_before, Args a) {
    typedef typename AccOf<T>::type A;
    constexpr int V = Width<T>::v;
    __shared__ A buffer[2][32];
    int turn = 0;
    rpb_pdl_trigger();
    rpb_pdl_wait();
    const A inv = A(1) / A(a.channels);
    A gwa[NV][V], gsc[NV][V], gwb[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) gwa[k][i] = gsc[k][i] = gwb[k][i] = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        Pack<T, V> up_[NV], zp[NV], rp[NV], op[NV], yp[NV], wa[NV], sc[NV], wb[NV];
        load_row<T, NV>(up_, u + row * a.u_row, a);
        load_row<T, NV>(zp, z ? z + row * a.z_row : nullptr, a);
        load_row<T, NV>(rp, r ? r + row * a.r_row : nullptr, a);
        load_row<T, NV>(op, dout ? dout + row * a.out_row : nullptr, a);
        load_row<T, NV>(yp, dy ? dy + row * a.y_row : nullptr, a);
        load_row<T, NV>(wa, w_after, a);
        load_row<T, NV>(sc, scale, a);
        load_row<T, NV>(wb, dy ? w_before : nullptr, a);
        A v[NV][V], sq = 0;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[k][i] = up(up_[k].v[i]);
                if (z) { const A g = up(zp[k].v[i]); v[k][i] *= g * logistic(g); }
                sq += v[k][i] * v[k][i];
            }
        const A i1 = w_after ? rsqrt_of(block_sum(sq, buffer, turn) * inv + A(a.eps_after)) : A(1);
        /* the gradient of out */
        A total[NV][V];
        if (dy) {
            A o[NV][V], dot = 0;
            sq = 0;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    A s = v[k][i] * i1;
                    if (w_after) s *= up(wa[k].v[i]);
                    if (scale) s *= up(sc[k].v[i]);
                    o[k][i] = up(rp[k].v[i]) + s;
                    sq += o[k][i] * o[k][i];
                    dot += up(yp[k].v[i]) * up(wb[k].v[i]) * o[k][i];
                }
            const A i2 = rsqrt_of(block_sum(sq, buffer, turn) * inv + A(a.eps_before));
            const A pull = block_sum(dot, buffer, turn) * inv * i2 * i2;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    gwb[k][i] += up(yp[k].v[i]) * o[k][i] * i2;
                    total[k][i] = up(op[k].v[i]) + i2 * (up(yp[k].v[i]) * up(wb[k].v[i]) - o[k][i] * pull);
                }
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) total[k][i] = up(op[k].v[i]);
        }
        A dot = 0;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = channel_of<V>(k), valid = a.channels - c;
            if (dr) {
                T* to = dr + row * a.dr_row + c;
                const Pack<T, V> have = acc_dr ? load_pack<T, V>(to, valid, a.vec) : zero_pack<T, V>();
                Pack<T, V> o;
#pragma unroll
                for (int i = 0; i < V; ++i) o.v[i] = down<T>(total[k][i] + up(have.v[i]));
                store_pack<T, V>(to, o, valid, a.vec);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const A t = v[k][i] * i1, w = w_after ? up(wa[k].v[i]) : A(1), s = scale ? up(sc[k].v[i]) : A(1);
                gwa[k][i] += total[k][i] * s * t;
                gsc[k][i] += total[k][i] * w * t;
                total[k][i] *= s * w;               /* now the gradient of t (of v where there is no norm) */
                dot += total[k][i] * v[k][i];
            }
        }
        const A pull = w_after ? block_sum(dot, buffer, turn) * inv * i1 * i1 : A(0);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = channel_of<V>(k), valid = a.channels - c;
            T *to_u = du ? du + row * a.du_row + c : nullptr, *to_z = dz ? dz + row * a.dz_row + c : nullptr;
            Pack<T, V> o = to_u && acc_du ? load_pack<T, V>(to_u, valid, a.vec) : zero_pack<T, V>();
            Pack<T, V> q = to_z && acc_dz ? load_pack<T, V>(to_z, valid, a.vec) : zero_pack<T, V>();
#pragma unroll
            for (int i = 0; i < V; ++i) {
                A dv = i1 * (total[k][i] - v[k][i] * pull);
                if (z) {
                    const A g = up(zp[k].v[i]), s = logistic(g);
                    q.v[i] = down<T>(up(q.v[i]) + dv * up(up_[k].v[i]) * s * (A(1) + g * (A(1) - s)));
                    dv *= g * s;
                }
                o.v[i] = down<T>(up(o.v[i]) + dv);
            }
            if (to_u) store_pack<T, V>(to_u, o, valid, a.vec);
            if (to_z) store_pack<T, V>(to_z, q, valid, a.vec);
        }
    }
    if (!parts) return;
    A* part = parts + (long long)blockIdx.x * 3 * a.channels;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = channel_of<V>(k);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (c + i < a.channels) {
                part[c + i] = gwa[k][i];
                part[a.channels + c + i] = gsc[k][i];
                part[2 * a.channels + c + i] = gwb[k][i];
            }
    }
}

/* packs per thread, and threads: the fewest packs that at most `most` threads cover the row with */
template <typename T> void shape_of(int channels, int most, int* packs, int* threads) {
    const int n = (channels + Width<T>::v - 1) / Width<T>::v;
    int p = 1;
    while ((n + p - 1) / p > most) p *= 2;
    *packs = p;
    *threads = ((n + p - 1) / p + 31) / 32 * 32;
}

/* Blocks of the backward call: each leaves one part of the weights' gradients behind. */
long long backward_blocks(const RpbBlockNorm* c) {
    const long long most = SM_COUNT * 4;
    return c->rows < most ? c->rows : most;
}

Args make_args(const RpbBlockNorm* c) {
    Args a;
    a.rows = c->rows; a.channels = c->channels; a.eps_after = c->eps_after; a.eps_before = c->eps_before;
    a.u_row = c->u_row; a.z_row = c->z_row; a.r_row = c->r_row; a.out_row = c->out_row; a.y_row = c->y_row;
    a.du_row = c->du_row; a.dz_row = c->dz_row; a.dr_row = c->dr_row;
    a.vec = true;
    return a;
}

/* rows as sequences of one row: a batch of `rows` */
Rows rows_of(const RpbBlockNorm* c, const void* p, long long row) { return {p, row, c->channels, c->channels}; }
int batch_of(const RpbBlockNorm* c) { return c->rows > 1 ? 2 : 1; }
template <typename T> bool whole(const RpbBlockNorm* c, const void* p, long long row) {
    return !p || aligned_rows(rows_of(c, p, row), batch_of(c), 1, sizeof(T), 16);
}

struct Operands { const void *u, *z, *w_after, *scale, *r, *w_before; };

template <typename T> bool weights_whole(const RpbBlockNorm* c, const Operands& o) {
    return whole<T>(c, o.u, c->u_row) && whole<T>(c, o.z, c->z_row) && whole<T>(c, o.r, c->r_row) && whole<T>(c, o.w_after, 0) &&
           whole<T>(c, o.scale, 0) && whole<T>(c, o.w_before, 0);
}

template <typename T, int NV>
int forward_n(void* out, void* y, const Operands& o, const RpbBlockNorm* c, int threads, cudaStream_t s) {
    Args a = make_args(c);
    a.vec = weights_whole<T>(c, o) && whole<T>(c, out, c->out_row) && whole<T>(c, y, c->y_row);
    const long long most = (long long)SM_COUNT * (2048 / threads) * 4;
    const unsigned blocks = (unsigned)(c->rows < most ? c->rows : most);
    SEQ_CUDA(rpb_launch(forward_kernel<T, NV>, dim3(blocks), dim3(threads), 0, s, 1, reinterpret_cast<T*>(out), reinterpret_cast<T*>(y),
                        reinterpret_cast<const T*>(o.u), reinterpret_cast<const T*>(o.z), reinterpret_cast<const T*>(o.w_after),
                        reinterpret_cast<const T*>(o.scale), reinterpret_cast<const T*>(o.r), reinterpret_cast<const T*>(o.w_before), a));
    rpb_count_launches(1);
    return 0;
}

struct Wanted { void *du, *dz, *dr, *dw_after, *dscale, *dw_before; int accumulate; };

template <typename T, int NV>
int backward_n(const Wanted& w, const void* dout, const void* dy, const Operands& o, void* ws, const RpbBlockNorm* c, int threads, cudaStream_t s) {
    typedef typename AccOf<T>::type A;
    Args a = make_args(c);
    a.vec = weights_whole<T>(c, o) && whole<T>(c, dout, c->out_row) && whole<T>(c, dy, c->y_row) && whole<T>(c, w.du, c->du_row) &&
            whole<T>(c, w.dz, c->dz_row) && whole<T>(c, w.dr, c->dr_row);
    const bool weights = w.dw_after || w.dscale || w.dw_before;
    const long long blocks = backward_blocks(c);
    SEQ_CUDA(rpb_launch(backward_kernel<T, NV>, dim3((unsigned)blocks), dim3(threads), 0, s, 1, reinterpret_cast<T*>(w.du), reinterpret_cast<T*>(w.dz),
                        reinterpret_cast<T*>(w.dr), weights ? reinterpret_cast<A*>(ws) : nullptr, (w.accumulate & RPB_NORM_ACC_DU) != 0,
                        (w.accumulate & RPB_NORM_ACC_DZ) != 0, (w.accumulate & RPB_NORM_ACC_DR) != 0, reinterpret_cast<const T*>(dout),
                        reinterpret_cast<const T*>(dy), reinterpret_cast<const T*>(o.u), reinterpret_cast<const T*>(o.z),
                        reinterpret_cast<const T*>(o.w_after), reinterpret_cast<const T*>(o.scale), reinterpret_cast<const T*>(o.r),
                        reinterpret_cast<const T*>(o.w_before), a));
    rpb_count_launches(1);
    if (!weights) return 0;
    const long long D = c->channels;
    PartSums d = {};
    d.out[0] = w.dw_after; d.first[0] = 0; d.accumulate[0] = (w.accumulate & RPB_NORM_ACC_DW_AFTER) != 0;
    d.out[1] = w.dscale; d.first[1] = D; d.accumulate[1] = (w.accumulate & RPB_NORM_ACC_DSCALE) != 0;
    d.out[2] = w.dw_before; d.first[2] = 2 * D; d.accumulate[2] = (w.accumulate & RPB_NORM_ACC_DW_BEFORE) != 0;
    d.cols[0] = d.cols[1] = d.cols[2] = D;
    return sum_parts<T>(d, ws, (int)blocks, 3 * D, s);
}

template <typename T> int run_forward(void* out, void* y, const Operands& o, const RpbBlockNorm* c, cudaStream_t s) {
    int packs, threads;
    shape_of<T>(c->channels, 512, &packs, &threads);
    switch (packs) {
        case 1: return forward_n<T, 1>(out, y, o, c, threads, s);
        case 2: return forward_n<T, 2>(out, y, o, c, threads, s);
        case 4: return forward_n<T, 4>(out, y, o, c, threads, s);
        case 8: return forward_n<T, 8>(out, y, o, c, threads, s);
        case 16: return forward_n<T, 16>(out, y, o, c, threads, s);
    }
    return -1;
}
template <typename T> int run_backward(const Wanted& w, const void* dout, const void* dy, const Operands& o, void* ws, const RpbBlockNorm* c, cudaStream_t s) {
    int packs, threads;
    shape_of<T>(c->channels, 512, &packs, &threads);
    switch (packs) {
        case 1: return backward_n<T, 1>(w, dout, dy, o, ws, c, threads, s);
        case 2: return backward_n<T, 2>(w, dout, dy, o, ws, c, threads, s);
        case 4: return backward_n<T, 4>(w, dout, dy, o, ws, c, threads, s);
        case 8: return backward_n<T, 8>(w, dout, dy, o, ws, c, threads, s);
        case 16: return backward_n<T, 16>(w, dout, dy, o, ws, c, threads, s);
    }
    return -1;
}

const char* bad_geometry(const RpbBlockNorm* c, DType dtype) {
    if (!c) return "no geometry";
    if (!rpb_dtype_size((int)dtype)) return "unknown element type";
    if (c->rows <= 0 || c->channels <= 0) return "rows and channels must be positive";
    if (c->channels > MAX_CHANNELS) return "rows longer than 16384 channels";
    if (!(c->eps_after >= 0) || !(c->eps_before >= 0)) return "eps must not be negative";
    return nullptr;
}
bool readable_rows(const RpbBlockNorm* c, const void* p, long long row) { return !p || c->rows == 1 || row >= 0; }
bool writable_rows(const RpbBlockNorm* c, const void* p, long long row) { return !p || c->rows == 1 || row >= c->channels; }
/* whether rows of two operands meet */
bool meet(const RpbBlockNorm* c, const void* p, long long p_row, const void* q, long long q_row, size_t es) {
    if (!p || !q) return false;
    const long long rows = c->rows < 0x7fffffffLL ? c->rows : 0x7fffffffLL;
    return overlaps({p, 0, p_row, c->channels}, {q, 0, q_row, c->channels}, 1, (int)rows, es);
}

}  // namespace rpb_norm

using namespace rpb_seq;
using namespace rpb_norm;

extern "C" {

void rpb_block_norm_packed(RpbBlockNorm* c, long long rows, int channels, float eps) {
    memset(c, 0, sizeof(*c));
    c->rows = rows; c->channels = channels; c->eps_after = c->eps_before = eps;
    c->u_row = c->z_row = c->r_row = c->out_row = c->y_row = c->du_row = c->dz_row = c->dr_row = channels;
}

int rp_block_norm_ex(void* out, void* y, const void* u, const void* z, const void* w_after, const void* scale, const void* r, const void* w_before,
                     const RpbBlockNorm* c, DType dtype, int device_id, void* stream) {
    const char* name = "rp_block_norm_ex";
    const char* why = bad_geometry(c, dtype);
    if (why) return refuse(name, why);
    if (!u) return refuse(name, "u is needed");
    if (!out && !y) return refuse(name, "neither out nor y is wanted");
    if (y && !w_before) return refuse(name, "y needs w_before");
    if (device_id < 0) return refuse(name, "needs a CUDA device (no CPU path in this library)");
    if (!readable_rows(c, u, c->u_row) || !readable_rows(c, z, c->z_row) || !readable_rows(c, r, c->r_row)) return refuse(name, "strides of an operand");
    if (!writable_rows(c, out, c->out_row) || !writable_rows(c, y, c->y_row)) return refuse(name, "strides of out or y");
    const size_t es = rpb_dtype_size((int)dtype);
    const Rows ins[3] = {{u, 0, c->u_row, 0}, {z, 0, c->z_row, 0}, {r, 0, c->r_row, 0}};
    for (const Rows& i : ins)
        if (meet(c, out, c->out_row, i.p, i.row, es) || meet(c, y, c->y_row, i.p, i.row, es)) return refuse(name, "out or y overlaps an operand");
    if (meet(c, out, c->out_row, y, c->y_row, es)) return refuse(name, "out and y overlap");
    DeviceScope scope;
    if (scope.enter(device_id)) return refuse(name, "no such device");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const Operands o = {u, z, w_after, scale, r, w_before};
    switch ((int)dtype) {
        case DTYPE_FLOAT32: return run_forward<float>(out, y, o, c, s);
        case DTYPE_FLOAT64: return run_forward<double>(out, y, o, c, s);
        case DTYPE_FLOAT16: return run_forward<__half>(out, y, o, c, s);
        case DTYPE_BFLOAT16: return run_forward<__nv_bfloat16>(out, y, o, c, s);
    }
    return -1;
}

long long rp_block_norm_ws_bytes(const RpbBlockNorm* c, DType dtype) {
    const char* why = bad_geometry(c, dtype);
    if (why) return refuse("rp_block_norm_ws_bytes", why);
    return backward_blocks(c) * 3 * c->channels * ((int)dtype == DTYPE_FLOAT64 ? 8 : 4);
}

int rp_block_norm_grad_ex(void* du, void* dz, void* dr, void* dw_after, void* dscale, void* dw_before, int accumulate, const void* dout, const void* dy,
                          const void* u, const void* z, const void* w_after, const void* scale, const void* r, const void* w_before, void* ws,
                          const RpbBlockNorm* c, DType dtype, int device_id, void* stream) {
    const char* name = "rp_block_norm_grad_ex";
    const char* why = bad_geometry(c, dtype);
    if (why) return refuse(name, why);
    if (!u) return refuse(name, "u is needed");
    if (!dout && !dy) return refuse(name, "neither dout nor dy is given");
    if (dy && !w_before) return refuse(name, "dy needs w_before");
    if (!du && !dz && !dr && !dw_after && !dscale && !dw_before) return refuse(name, "no gradient is wanted");
    if ((dz && !z) || (dw_after && !w_after) || (dscale && !scale) || (dw_before && !dy)) return refuse(name, "a gradient of an operand that is not given");
    if ((dw_after || dscale || dw_before) && !ws) return refuse(name, "the weights' gradients need a workspace");
    if (device_id < 0) return refuse(name, "needs a CUDA device (no CPU path in this library)");
    const Rows ins[5] = {{u, 0, c->u_row, 0}, {z, 0, c->z_row, 0}, {r, 0, c->r_row, 0}, {dout, 0, c->out_row, 0}, {dy, 0, c->y_row, 0}};
    const Rows outs[3] = {{du, 0, c->du_row, 0}, {dz, 0, c->dz_row, 0}, {dr, 0, c->dr_row, 0}};
    const size_t es = rpb_dtype_size((int)dtype);
    for (const Rows& i : ins)
        if (!readable_rows(c, i.p, i.row)) return refuse(name, "strides of an operand");
    for (int k = 0; k < 3; ++k) {
        if (!writable_rows(c, outs[k].p, outs[k].row)) return refuse(name, "strides of a gradient");
        for (const Rows& i : ins)
            if (meet(c, outs[k].p, outs[k].row, i.p, i.row, es)) return refuse(name, "a gradient overlaps an operand");
        for (int j = 0; j < k; ++j)
            if (meet(c, outs[k].p, outs[k].row, outs[j].p, outs[j].row, es)) return refuse(name, "two gradients overlap");
    }
    DeviceScope scope;
    if (scope.enter(device_id)) return refuse(name, "no such device");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const Operands o = {u, z, w_after, scale, r, w_before};
    const Wanted w = {du, dz, dr, dw_after, dscale, dw_before, accumulate};
    switch ((int)dtype) {
        case DTYPE_FLOAT32: return run_backward<float>(w, dout, dy, o, ws, c, s);
        case DTYPE_FLOAT64: return run_backward<double>(w, dout, dy, o, ws, c, s);
        case DTYPE_FLOAT16: return run_backward<__half>(w, dout, dy, o, ws, c, s);
        case DTYPE_BFLOAT16: return run_backward<__nv_bfloat16>(w, dout, dy, o, ws, c, s);
    }
    return -1;
}

}  // extern "C"
