/*
 * The norms around a block, with its gate and the scaled add to the residual, one pass over each row:
 *   v = u z / (1 + exp(-z)) (or u),  s = v rsqrt(mean v^2 + eps_after) w_after (or v),  out = r + scale s,
 *   y = out rsqrt(mean out^2 + eps_before) w_before.
 * Backward: with t = v i (i = rsqrt(mean v^2 + eps)) and m the gradient of t, dv = i (m - t mean(m t)); y's norm likewise.
 * A block of threads holds a whole row in registers, so each operand is read once and the row's sums are taken from there.
 * Its floor is memory (51 us for the forward call at 8192 x 4096 bf16); it takes 84 us there, for the latency of two block sums per row,
 * and 100 us for the backward call at 4001 x 2999 f16, with three (there the forward call's issue slots are 68% busy, the backward
 * call's 50%).  Rows of up to 256 16-bit channels have a block of one warp each, of which too few run at once: 37 us at 32768 x 128
 * bf16 against 6, and 260 us forward and backward against 13.
 */
#include "seq_common.cuh"

namespace rpb_norm {

using namespace rpb_seq;

constexpr int MAX_CHANNELS = 8192;

struct Args {
    long long rows;
    int channels, classes;      /* rows r, r + classes, ... begin at the same offset from a 16-byte boundary */
    double eps_after, eps_before;
    int u_row, z_row, r_row, out_row, y_row, du_row, dz_row, dr_row;        /* below 2^31; their products with a row are 64 bits */
};

template <typename T> struct Width { static constexpr int v = 16 / sizeof(T); };

__device__ __forceinline__ float rsqrt_of(float v) { return rsqrtf(v); }
__device__ __forceinline__ double rsqrt_of(double v) { return rsqrt(v); }

/* Sums over the block of N values per thread; every thread gets them.  The two halves of the buffer take turns, so that one
 * barrier is enough: a half is written again only behind the next sum's barrier. */
template <int N, typename A> __device__ __forceinline__ void block_sums(A (&v)[N], A (*buffer)[N][32], int& turn) {
#pragma unroll
    for (int m = 16; m >= 1; m /= 2)
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] += __shfl_xor_sync(0xffffffffu, v[j], m);
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (warps == 1) return;
    A (*slots)[32] = buffer[turn];
    turn ^= 1;
    if (lane == 0)
#pragma unroll
        for (int j = 0; j < N; ++j) slots[j][threadIdx.x >> 5] = v[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = lane < warps ? slots[j][lane] : A(0);
#pragma unroll
    for (int m = 16; m >= 1; m /= 2)
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] += __shfl_xor_sync(0xffffffffu, v[j], m);
}

/* A thread's channels: NV packs of V.  PACKS: pack k lies on a 16-byte boundary of the row, at channel (k threads + thread) V
 * minus the row's offset from such a boundary (the first and the last pack may stick out of the row); else value i of pack k is
 * channel (k V + i) threads + thread, so that a warp's single values are neighbours. */
template <typename T, int NV, bool PACKS> struct Span {
    static constexpr int V = Width<T>::v;
    static constexpr unsigned ALL = (1u << V) - 1;
    int base, step;
    unsigned mask[NV];          /* which values of a pack are channels of the row */
    int bytes[NV];              /* of a pack up to the row's end */
    int off;                    /* channels that the first pack begins in front of the row */
    __device__ __forceinline__ Span(const T* row, int channels) {
        off = PACKS ? (int)(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T)) : 0;
        base = PACKS ? (int)threadIdx.x * V - off : (int)threadIdx.x;
        step = PACKS ? (int)blockDim.x * V : (int)blockDim.x;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            mask[k] = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = channel(k, i);
                if (c >= 0 && c < channels) mask[k] |= 1u << i;
            }
            const int left = channels - channel(k, 0);
            bytes[k] = (int)sizeof(T) * (left < 0 ? 0 : left > V ? V : left);
        }
    }
    __device__ __forceinline__ int channel(int k, int i) const { return PACKS ? base + k * step + i : base + (k * V + i) * step; }
    __device__ __forceinline__ bool has(int k, int i) const { return mask[k] >> i & 1; }
    /* The thread's packs of a row into its slots, which nobody else reads, asynchronously where they lie on boundaries.  A pack
     * that begins in front of the row brings the end of the row before along (take() leaves it out); the operand's first row,
     * with nothing in front of it, is read value by value, as are rows off the boundaries. */
    __device__ __forceinline__ void bring(Pack<T, V>* slots, const T* row, bool given, bool first) const {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            Pack<T, V>* to = slots + k * blockDim.x + threadIdx.x;
            if (PACKS && !(first && off)) {
                async_copy_part<16>(to, row + channel(k, 0), given ? bytes[k] : 0);
            } else {
                Pack<T, V> p = zero_pack<T, V>();
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (given && has(k, i)) p.v[i] = row[channel(k, i)];
                *to = p;
            }
        }
    }
    __device__ __forceinline__ Pack<T, V> take(const Pack<T, V>* slots, int k) const {
        Pack<T, V> p = slots[k * blockDim.x + threadIdx.x];
        if (PACKS && off && k == 0 && threadIdx.x == 0) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (!has(k, i)) p.v[i] = down<T>(typename AccOf<T>::type(0));
        }
        return p;
    }
    __device__ __forceinline__ Pack<T, V> load_one(const T* row, int k) const {
        Pack<T, V> p = zero_pack<T, V>();
        if (PACKS && mask[k] == ALL) return *reinterpret_cast<const Pack<T, V>*>(row + channel(k, 0));
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (has(k, i)) p.v[i] = row[channel(k, i)];
        return p;
    }
    /* The thread's channels of a weight: packs lie on boundaries of the row, which need not be boundaries of the weight. */
    __device__ __forceinline__ Pack<T, V> load_weight(const T* w, int k) const {
        if (PACKS && mask[k] == ALL && reinterpret_cast<uintptr_t>(w + channel(k, 0)) % 16 == 0)
            return *reinterpret_cast<const Pack<T, V>*>(w + channel(k, 0));
        Pack<T, V> p = zero_pack<T, V>();
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (has(k, i)) p.v[i] = w[channel(k, i)];
        return p;
    }
    __device__ __forceinline__ void store(T* row, int k, const Pack<T, V>& p) const {
        if (PACKS && mask[k] == ALL) { *reinterpret_cast<Pack<T, V>*>(row + channel(k, 0)) = p; return; }
        if (PACKS && mask[k] == 0) return;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (has(k, i)) row[channel(k, i)] = p.v[i];
    }
};

/* The weights of a thread's channels stay in shared memory as the thread needs them. */
template <typename T> __device__ __forceinline__ Pack<T, Width<T>::v>* weight_slots() {
    extern __shared__ __align__(16) unsigned char raw_shared[];
    return reinterpret_cast<Pack<T, Width<T>::v>*>(raw_shared);
}
template <typename T, int NV, bool PACKS>
__device__ __forceinline__ void keep_weights(Pack<T, Width<T>::v>* slots, const T* w, const Span<T, NV, PACKS>& span) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        Pack<T, Width<T>::v> p = zero_pack<T, Width<T>::v>();
#pragma unroll
        for (int i = 0; i < Width<T>::v; ++i)
            if (w && span.has(k, i)) p.v[i] = w[span.channel(k, i)];
        slots[k * blockDim.x + threadIdx.x] = p;
    }
}

/* Block b takes the rows of class b % classes, every (gridDim / classes)-th of them. */
struct Turn { long long row, step; };
__device__ __forceinline__ Turn turn_of(const Args& a) {
    const int per_class = gridDim.x / a.classes;
    return {(long long)(blockIdx.x / a.classes) * a.classes + blockIdx.x % a.classes, (long long)per_class * a.classes};
}

/* Rows of a block in shared memory: the one worked on and the next two or one; 0 for rows too wide for that (over 1024 packs),
 * whose values are read where they lie each time they are needed. */
template <int NV> struct Slots { static constexpr int forward = NV <= 2 ? 3 : 0, backward = NV == 1 ? 3 : NV == 2 ? 2 : 0; };

template <typename T, int NV, bool PACKS>
__global__ void __launch_bounds__(512, NV == 1 ? 2 : 1)
forward_kernel(T* __restrict__ out, T* __restrict__ y, const T* __restrict__ u, const T* __restrict__ z, const T* __restrict__ w_after,
               const T* __restrict__ scale, const T* __restrict__ r, const T* __restrict__ w_before, Args a) {
    typedef typename AccOf<T>::type A;
    constexpr int V = Width<T>::v, SLOTS = Slots<NV>::forward;
    __shared__ A buffer[2][1][32];
    int turn = 0;
    rpb_pdl_trigger();
    rpb_pdl_wait();
    const A inv = A(1) / A(a.channels);
    const Turn t = turn_of(a);
    if (t.row >= a.rows) return;
    const Span<T, NV, PACKS> span(u + t.row * a.u_row, a.channels);
    const int nt = blockDim.x, tid = threadIdx.x, per = NV * nt;
    Pack<T, V> *ws = weight_slots<T>(), *ring = ws + 3 * per;
    auto fetch = [&](long long row, int slot) {
        const bool in = row < a.rows;
        Pack<T, V>* to = ring + slot * 3 * per;
        span.bring(to, u + (long long)(int)row * a.u_row, in, row == 0);
        if (z) span.bring(to + per, z + (long long)(int)row * a.z_row, in, row == 0);
        if (r) span.bring(to + 2 * per, r + (long long)(int)row * a.r_row, in, row == 0);
        async_commit();
    };
#pragma unroll
    for (int k = 0; k + 1 < SLOTS; ++k) fetch(t.row + k * t.step, k);
    if (SLOTS) {
    keep_weights(ws, w_after, span);
    keep_weights(ws + per, scale, span);
    keep_weights(ws + 2 * per, w_before, span);
    }
    int slot = 0;
    for (long long row = t.row; row < a.rows; row += t.step) {
        if (SLOTS) async_wait<SLOTS ? SLOTS - 2 : 0>();
        const Pack<T, V>* from = ring + slot * 3 * per;
        const T* rows[3] = {u + (long long)(int)row * a.u_row, z + (long long)(int)row * a.z_row, r + (long long)(int)row * a.r_row};
        auto take = [&](int n, int k) { return SLOTS ? span.take(from + n * per, k) : span.load_one(rows[n], k); };
        auto weight = [&](int n, const T* w, int k) { return SLOTS ? ws[n * per + k * nt + tid] : w ? span.load_weight(w, k) : zero_pack<T, V>(); };
        A o[NV][V], sq[1] = {0};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const Pack<T, V> up_ = take(0, k), zp = z ? take(1, k) : up_;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                o[k][i] = up(up_.v[i]);
                if (z) { const A g = up(zp.v[i]); o[k][i] *= g * logistic(g); }
                sq[0] += o[k][i] * o[k][i];
            }
        }
        if (SLOTS) fetch(row + (SLOTS - 1) * t.step, slot == 0 ? SLOTS - 1 : slot - 1);
        A i1 = 1;
        if (w_after) {
            block_sums(sq, buffer, turn);
            i1 = rsqrt_of(sq[0] * inv + A(a.eps_after));
        }
        sq[0] = 0;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const Pack<T, V> wp = weight(0, w_after, k), sp = weight(1, scale, k);
            if (w_after) {
#pragma unroll
                for (int i = 0; i < V; ++i) o[k][i] = o[k][i] * i1 * up(wp.v[i]);
            }
            if (scale) {
#pragma unroll
                for (int i = 0; i < V; ++i) o[k][i] *= up(sp.v[i]);
            }
            if (r) {
                const Pack<T, V> rp = take(2, k);
#pragma unroll
                for (int i = 0; i < V; ++i) o[k][i] += up(rp.v[i]);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) sq[0] += o[k][i] * o[k][i];
            if (out) span.store(out + (long long)(int)row * a.out_row, k, store_form<T, V>(o[k]));
        }
        if (y) {
            block_sums(sq, buffer, turn);
            const A i2 = rsqrt_of(sq[0] * inv + A(a.eps_before));
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const Pack<T, V> wp = weight(2, w_before, k);
                A q[V];
#pragma unroll
                for (int i = 0; i < V; ++i) q[i] = o[k][i] * i2 * up(wp.v[i]);
                span.store(y + (long long)(int)row * a.y_row, k, store_form<T, V>(q));
            }
        }
        slot = slot + 1 >= SLOTS ? 0 : slot + 1;
    }
    async_wait<0>();
}

/* Each block keeps its part of the weights' gradients in registers; sum_parts adds the blocks' parts [3][channels]: w_after,
 * scale, w_before. */
template <typename T, int NV, bool PACKS>
__global__ void __launch_bounds__(512)
backward_kernel(T* du, T* dz, T* dr, typename AccOf<T>::type* __restrict__ parts, int acc_du, int acc_dz, int acc_dr, const T* __restrict__ dout,
                const T* __restrict__ dy, const T* __restrict__ u, const T* __restrict__ z, const T* __restrict__ w_after, const T* __restrict__ scale,
                const T* __restrict__ r, const T* __restrict__ w_before, Args a) {
    typedef typename AccOf<T>::type A;
    constexpr int V = Width<T>::v, SLOTS = Slots<NV>::backward;
    __shared__ A buffer[2][2][32];
    int turn = 0;
    rpb_pdl_trigger();
    rpb_pdl_wait();
    const A inv = A(1) / A(a.channels);
    const Turn t = turn_of(a);
    const int nt = blockDim.x, tid = threadIdx.x, per = NV * nt;
    const Span<T, NV, PACKS> span(u + t.row * a.u_row, a.channels);
    Pack<T, V> *ws = weight_slots<T>(), *ring = ws + 3 * per;
    auto fetch = [&](long long row, int slot) {
        const bool in = row < a.rows;
        Pack<T, V>* to = ring + slot * 5 * per;
        span.bring(to, u + (long long)(int)row * a.u_row, in, row == 0);
        if (z) span.bring(to + per, z + (long long)(int)row * a.z_row, in, row == 0);
        if (r) span.bring(to + 2 * per, r + (long long)(int)row * a.r_row, in, row == 0);
        if (dout) span.bring(to + 3 * per, dout + (long long)(int)row * a.out_row, in, row == 0);
        if (dy) span.bring(to + 4 * per, dy + (long long)(int)row * a.y_row, in, row == 0);
        async_commit();
    };
#pragma unroll
    for (int k = 0; k + 1 < SLOTS; ++k) fetch(t.row + k * t.step, k);
    if (SLOTS) {
    keep_weights(ws, w_after, span);
    keep_weights(ws + per, scale, span);
    keep_weights(ws + 2 * per, dy ? w_before : nullptr, span);
    }
    A gwa[NV][V], gsc[NV][V], gwb[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) gwa[k][i] = gsc[k][i] = gwb[k][i] = 0;
    int slot = 0;
    for (long long row = t.row; row < a.rows; row += t.step) {
        if (SLOTS) async_wait<SLOTS ? SLOTS - 2 : 0>();
        const Pack<T, V>* from = ring + slot * 5 * per;
        const T* rows[5] = {u + (long long)(int)row * a.u_row, z + (long long)(int)row * a.z_row, r + (long long)(int)row * a.r_row, dout + (long long)(int)row * a.out_row, dy + (long long)(int)row * a.y_row};
        auto take = [&](int n, int k) { return SLOTS ? span.take(from + n * per, k) : span.load_one(rows[n], k); };
        auto weight = [&](int n, const T* w, int k) { return SLOTS ? ws[n * per + k * nt + tid] : w ? span.load_weight(w, k) : zero_pack<T, V>(); };
        A v[NV][V], total[NV][V], sq[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const Pack<T, V> up_ = take(0, k), zp = z ? take(1, k) : up_;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[k][i] = up(up_.v[i]);
                if (z) { const A g = up(zp.v[i]); v[k][i] *= g * logistic(g); }
                sq[0] += v[k][i] * v[k][i];
            }
        }
        if (SLOTS) fetch(row + (SLOTS - 1) * t.step, slot == 0 ? SLOTS - 1 : slot - 1);
        A i1 = 1;
        if (w_after) {
            block_sums(sq, buffer, turn);
            i1 = rsqrt_of(sq[0] * inv + A(a.eps_after));
        }
        /* total: the gradient of out */
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) total[k][i] = 0;
        if (dy) {
            sq[0] = sq[1] = 0;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const Pack<T, V> wa = weight(0, w_after, k), sc = weight(1, scale, k), wb = weight(2, dy ? w_before : nullptr, k), yp = take(4, k);
#pragma unroll
                for (int i = 0; i < V; ++i) total[k][i] = v[k][i] * i1;         /* out itself, for now */
                if (w_after) {
#pragma unroll
                    for (int i = 0; i < V; ++i) total[k][i] *= up(wa.v[i]);
                }
                if (scale) {
#pragma unroll
                    for (int i = 0; i < V; ++i) total[k][i] *= up(sc.v[i]);
                }
                if (r) {
                    const Pack<T, V> rp = take(2, k);
#pragma unroll
                    for (int i = 0; i < V; ++i) total[k][i] += up(rp.v[i]);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    sq[0] += total[k][i] * total[k][i];
                    sq[1] += up(yp.v[i]) * up(wb.v[i]) * total[k][i];
                }
            }
            block_sums(sq, buffer, turn);
            const A i2 = rsqrt_of(sq[0] * inv + A(a.eps_before)), pull = sq[1] * inv * i2 * i2;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const Pack<T, V> wb = weight(2, dy ? w_before : nullptr, k), yp = take(4, k);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const A o = total[k][i], g = up(yp.v[i]);
                    gwb[k][i] += g * o * i2;
                    total[k][i] = i2 * (g * up(wb.v[i]) - o * pull);
                }
            }
        }
        sq[0] = sq[1] = 0;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (dout) {
                const Pack<T, V> op = take(3, k);
#pragma unroll
                for (int i = 0; i < V; ++i) total[k][i] += up(op.v[i]);
            }
            if (dr) {
                T* to = dr + (long long)(int)row * a.dr_row;
                A sum[V];
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] = total[k][i];
                if (acc_dr) {
                    const Pack<T, V> have = span.load_one(to, k);
#pragma unroll
                    for (int i = 0; i < V; ++i) sum[i] += up(have.v[i]);
                }
                span.store(to, k, store_form<T, V>(sum));
            }
            const Pack<T, V> wa = weight(0, w_after, k), sc = weight(1, scale, k);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const A m = v[k][i] * i1, w = w_after ? up(wa.v[i]) : A(1), s = scale ? up(sc.v[i]) : A(1);
                gwa[k][i] += total[k][i] * s * m;
                gsc[k][i] += total[k][i] * w * m;
                total[k][i] *= s * w;               /* now the gradient of v i1 (of v where there is no norm) */
                sq[0] += total[k][i] * v[k][i];
            }
        }
        A pull = 0;
        if (w_after) {
            block_sums(sq, buffer, turn);
            pull = sq[0] * inv * i1 * i1;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            A gu[V], gz[V];
#pragma unroll
            for (int i = 0; i < V; ++i) gu[i] = i1 * (total[k][i] - v[k][i] * pull);
            if (z) {
                const Pack<T, V> up_ = take(0, k), zp = take(1, k);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const A g = up(zp.v[i]), s = logistic(g);
                    gz[i] = gu[i] * up(up_.v[i]) * s * (A(1) + g * (A(1) - s));
                    gu[i] *= g * s;
                }
            }
            if (du) {
                T* to = du + (long long)(int)row * a.du_row;
                if (acc_du) {
                    const Pack<T, V> have = span.load_one(to, k);
#pragma unroll
                    for (int i = 0; i < V; ++i) gu[i] += up(have.v[i]);
                }
                span.store(to, k, store_form<T, V>(gu));
            }
            if (dz && z) {
                T* to = dz + (long long)(int)row * a.dz_row;
                if (acc_dz) {
                    const Pack<T, V> have = span.load_one(to, k);
#pragma unroll
                    for (int i = 0; i < V; ++i) gz[i] += up(have.v[i]);
                }
                span.store(to, k, store_form<T, V>(gz));
            }
        }
        slot = slot + 1 >= SLOTS ? 0 : slot + 1;
    }
    async_wait<0>();
    if (!parts) return;
    A* part = parts + (long long)blockIdx.x * 3 * a.channels;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (span.has(k, i)) {
                const int c = span.channel(k, i);
                part[c] = gwa[k][i];
                part[a.channels + c] = gsc[k][i];
                part[2 * a.channels + c] = gwb[k][i];
            }
}

/* packs per thread, and threads: the fewest packs that at most 512 threads cover the row with; `spare`: rows that begin between
 * two 16-byte boundaries stick out into one pack more */
template <typename T> void shape_of(int channels, bool spare, int* packs, int* threads) {
    constexpr int most[] = {1, 2, sizeof(T) == 2 ? 3 : 4, sizeof(T) == 4 ? 5 : 8, 9};
    const int n = (channels + Width<T>::v - 1) / Width<T>::v + spare;
    int i = 0;
    while ((n + most[i] - 1) / most[i] > 512) ++i;
    *packs = most[i];
    *threads = ((n + most[i] - 1) / most[i] + 31) / 32 * 32;
}

/* Blocks of the backward call: each leaves one part of the weights' gradients behind.  A multiple of 8, so that the classes of
 * rows (8 at most) share them evenly. */
long long backward_blocks(const RpbBlockNorm* c) {
    /* what the registers hold at once of blocks of 256 threads and more; of narrower ones they would hold more */
    const long long most = c->channels > 2048 ? SM_COUNT / 8 * 8 : SM_COUNT * 2;
    const long long rows = (c->rows + 7) / 8 * 8;
    return rows < most ? rows : most;
}

struct Operand { const void* p; long long row; };

/* Whether the rows can be moved in packs, and how many rows on they begin at the same offset from a 16-byte boundary: all
 * operands must have their rows at the same offsets. */
template <typename T> bool packs_of(const RpbBlockNorm* c, const Operand* o, int n, int* classes) {
    constexpr int V = Width<T>::v;
    const uintptr_t at = reinterpret_cast<uintptr_t>(o[0].p) % 16;
    if (at % sizeof(T)) return false;
    for (int i = 1; i < n; ++i) {
        if (!o[i].p) continue;
        if (reinterpret_cast<uintptr_t>(o[i].p) % 16 != at) return false;
        if (c->rows > 1 && (o[i].row - o[0].row) % V != 0) return false;
    }
    int k = 1;
    while (c->rows > 1 && o[0].row * k % V != 0) k *= 2;
    /* rows off the boundaries: their first pack reaches up to V - 1 channels in front of the row, which the row before must hold */
    if (k > 1 || at != 0)
        for (int i = 0; i < n; ++i)
            if (o[i].p && c->rows > 1 && o[i].row < V) return false;
    *classes = k;
    return true;
}

Args make_args(const RpbBlockNorm* c) {
    Args a;
    a.rows = c->rows; a.channels = c->channels; a.classes = 1; a.eps_after = c->eps_after; a.eps_before = c->eps_before;
    a.u_row = (int)c->u_row; a.z_row = (int)c->z_row; a.r_row = (int)c->r_row; a.out_row = (int)c->out_row; a.y_row = (int)c->y_row;
    a.du_row = (int)c->du_row; a.dz_row = (int)c->dz_row; a.dr_row = (int)c->dr_row;
    return a;
}

struct Operands { const void *u, *z, *w_after, *scale, *r, *w_before; };

template <typename T, int NV, bool PACKS>
int forward_n(void* out, void* y, const Operands& o, const Args& a, int threads, cudaStream_t s) {
    const size_t smem = Slots<NV>::forward ? (size_t)(3 + Slots<NV>::forward * 3) * NV * threads * 16 : 0;
    static unsigned char done[64];
    int device = 0;
    SEQ_CUDA(cudaGetDevice(&device));
    if (allow_shared(forward_kernel<T, NV, PACKS>, smem, device, done)) return -1;
    /* as many blocks as the chip holds at once, at least one row each; a multiple of 8 for the classes */
    long long most = (long long)SM_COUNT * (NV > 1 ? 1 : 1024 / threads < 8 ? 1024 / threads : 8);
    most -= most % 8;
    const long long rows = (a.rows + 7) / 8 * 8;
    const unsigned blocks = (unsigned)(rows < most ? rows : most);
    SEQ_CUDA(rpb_launch(forward_kernel<T, NV, PACKS>, dim3(blocks), dim3(threads), smem, s, 1, reinterpret_cast<T*>(out), reinterpret_cast<T*>(y),
                        reinterpret_cast<const T*>(o.u), reinterpret_cast<const T*>(o.z), reinterpret_cast<const T*>(o.w_after),
                        reinterpret_cast<const T*>(o.scale), reinterpret_cast<const T*>(o.r), reinterpret_cast<const T*>(o.w_before), a));
    rpb_count_launches(1);
    return 0;
}

struct Wanted { void *du, *dz, *dr, *dw_after, *dscale, *dw_before; int accumulate; };

template <typename T, int NV, bool PACKS>
int backward_n(const Wanted& w, const void* dout, const void* dy, const Operands& o, void* ws, const Args& a, long long blocks, int threads,
               cudaStream_t s) {
    typedef typename AccOf<T>::type A;
    const bool weights = w.dw_after || w.dscale || w.dw_before;
    const size_t smem = Slots<NV>::backward ? (size_t)(3 + Slots<NV>::backward * 5) * NV * threads * 16 : 0;
    static unsigned char done[64];
    int device = 0;
    SEQ_CUDA(cudaGetDevice(&device));
    if (allow_shared(backward_kernel<T, NV, PACKS>, smem, device, done)) return -1;
    SEQ_CUDA(rpb_launch(backward_kernel<T, NV, PACKS>, dim3((unsigned)blocks), dim3(threads), smem, s, 1, reinterpret_cast<T*>(w.du),
                        reinterpret_cast<T*>(w.dz), reinterpret_cast<T*>(w.dr), weights ? reinterpret_cast<A*>(ws) : nullptr,
                        (w.accumulate & RPB_NORM_ACC_DU) != 0, (w.accumulate & RPB_NORM_ACC_DZ) != 0, (w.accumulate & RPB_NORM_ACC_DR) != 0,
                        reinterpret_cast<const T*>(dout), reinterpret_cast<const T*>(dy), reinterpret_cast<const T*>(o.u), reinterpret_cast<const T*>(o.z),
                        reinterpret_cast<const T*>(o.w_after), reinterpret_cast<const T*>(o.scale), reinterpret_cast<const T*>(o.r),
                        reinterpret_cast<const T*>(o.w_before), a));
    rpb_count_launches(1);
    if (!weights) return 0;
    const long long D = a.channels;
    PartSums d = {};
    d.out[0] = w.dw_after; d.first[0] = 0; d.accumulate[0] = (w.accumulate & RPB_NORM_ACC_DW_AFTER) != 0;
    d.out[1] = w.dscale; d.first[1] = D; d.accumulate[1] = (w.accumulate & RPB_NORM_ACC_DSCALE) != 0;
    d.out[2] = w.dw_before; d.first[2] = 2 * D; d.accumulate[2] = (w.accumulate & RPB_NORM_ACC_DW_BEFORE) != 0;
    d.cols[0] = d.cols[1] = d.cols[2] = D;
    return sum_parts<T>(d, ws, (int)blocks, 3 * D, s);
}

/* The pack that rows between two boundaries need beyond the longest row is there only where rows are moved in packs. */
template <typename T, typename F> int by_packs(int packs, bool whole, F f) {
#define CASE(n) if (packs == n) return whole ? f(std::integral_constant<int, n>(), std::true_type()) : f(std::integral_constant<int, n>(), std::false_type());
#define SPARE(n) if (packs == n && whole) return f(std::integral_constant<int, n>(), std::true_type());
    CASE(1) CASE(2)
    if constexpr (sizeof(T) == 2) { SPARE(3) }
    if constexpr (sizeof(T) == 4) { CASE(4) SPARE(5) }
    if constexpr (sizeof(T) == 8) { CASE(4) CASE(8) SPARE(9) }
#undef SPARE
#undef CASE
    return -1;
}

template <typename T> int run_forward(void* out, void* y, const Operands& o, const RpbBlockNorm* c, cudaStream_t s) {
    int packs, threads;
    Args a = make_args(c);
    const Operand rows[5] = {{o.u, c->u_row}, {o.z, c->z_row}, {o.r, c->r_row}, {out, c->out_row}, {y, c->y_row}};
    const bool whole = packs_of<T>(c, rows, 5, &a.classes);
    shape_of<T>(c->channels, whole && (a.classes > 1 || reinterpret_cast<uintptr_t>(o.u) % 16), &packs, &threads);
    return by_packs<T>(packs, whole, [&](auto n, auto p) { return forward_n<T, decltype(n)::value, decltype(p)::value>(out, y, o, a, threads, s); });
}
template <typename T> int run_backward(const Wanted& w, const void* dout, const void* dy, const Operands& o, void* ws, const RpbBlockNorm* c, cudaStream_t s) {
    int packs, threads;
    Args a = make_args(c);
    const Operand rows[8] = {{o.u, c->u_row}, {o.z, c->z_row}, {o.r, c->r_row}, {dout, c->out_row}, {dy, c->y_row}, {w.du, c->du_row},
                             {w.dz, c->dz_row}, {w.dr, c->dr_row}};
    const bool whole = packs_of<T>(c, rows, 8, &a.classes);
    shape_of<T>(c->channels, whole && (a.classes > 1 || reinterpret_cast<uintptr_t>(o.u) % 16), &packs, &threads);
    return by_packs<T>(packs, whole, [&](auto n, auto p) {
        return backward_n<T, decltype(n)::value, decltype(p)::value>(w, dout, dy, o, ws, a, backward_blocks(c), threads, s);
    });
}

const char* bad_geometry(const RpbBlockNorm* c, DType dtype) {
    if (!c) return "no geometry";
    if (!rpb_dtype_size((int)dtype)) return "unknown element type";
    if (c->rows <= 0 || c->channels <= 0) return "rows and channels must be positive";
    if (c->channels > MAX_CHANNELS) return "rows longer than 8192 channels";
    const long long strides[8] = {c->u_row, c->z_row, c->r_row, c->out_row, c->y_row, c->du_row, c->dz_row, c->dr_row};
    for (long long r : strides)
        if (c->rows > 0x7fffffffLL || r > 0x7fffffffLL || r < -0x7fffffffLL) return "rows and row strides must be below 2^31";
    if (!(c->eps_after >= 0) || !(c->eps_before >= 0)) return "eps must not be negative";
    return nullptr;
}
bool readable_rows(const RpbBlockNorm* c, const void* p, long long row) { return !p || c->rows == 1 || row >= 0; }
bool writable_rows(const RpbBlockNorm* c, const void* p, long long row) { return !p || c->rows == 1 || row >= c->channels; }
Area row_area(const RpbBlockNorm* c, const char* name, const void* p, long long row, size_t es) {
    return strided(name, {p, 0, row, c->channels}, 1, (int)c->rows, es);
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
    const long long D = c->channels;
    const Area outs[] = {row_area(c, "out", out, c->out_row, es), row_area(c, "y", y, c->y_row, es)};
    const Area ins[] = {row_area(c, "u", u, c->u_row, es), row_area(c, "z", z, c->z_row, es), row_area(c, "r", r, c->r_row, es),
                        packed("w_after", w_after, D, es), packed("scale", scale, D, es), packed("w_before", w_before, D, es)};
    if (refuse_buffers(name, outs, ins)) return -1;
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
    if (!readable_rows(c, u, c->u_row) || !readable_rows(c, z, c->z_row) || !readable_rows(c, r, c->r_row) || !readable_rows(c, dout, c->out_row) ||
        !readable_rows(c, dy, c->y_row))
        return refuse(name, "strides of an operand");
    if (!writable_rows(c, du, c->du_row) || !writable_rows(c, dz, c->dz_row) || !writable_rows(c, dr, c->dr_row)) return refuse(name, "strides of a gradient");
    const size_t es = rpb_dtype_size((int)dtype), as = dtype == DTYPE_FLOAT64 ? 8 : 4;
    const long long D = c->channels;
    const bool weights = dw_after || dscale || dw_before;
    const Area outs[] = {row_area(c, "du", du, c->du_row, es), row_area(c, "dz", dz, c->dz_row, es), row_area(c, "dr", dr, c->dr_row, es),
                         packed("dw_after", dw_after, D, es), packed("dscale", dscale, D, es), packed("dw_before", dw_before, D, es),
                         packed("ws", weights ? ws : nullptr, weights ? rp_block_norm_ws_bytes(c, dtype) / (long long)as : 0, as)};
    const Area ins[] = {row_area(c, "u", u, c->u_row, es), row_area(c, "z", z, c->z_row, es), row_area(c, "r", r, c->r_row, es),
                        row_area(c, "dout", dout, c->out_row, es), row_area(c, "dy", dy, c->y_row, es),
                        packed("w_after", w_after, D, es), packed("scale", scale, D, es), packed("w_before", w_before, D, es)};
    if (refuse_buffers(name, outs, ins)) return -1;
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
