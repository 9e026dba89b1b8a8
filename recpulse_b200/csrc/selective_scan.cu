/*
 * Selective state space scan: per sequence and channel a vector h of `states` values with
 *   delta = dt + dt_bias (behind a softplus when asked for),   h_t = exp(delta A) h_{t-1} + delta x_t B_t,
 *   y_t = C_t . h_t + D x_t,   out = y (or y z / (1 + exp(-z))).
 * B and C are shared by the channels of a group.  One exponential per row, channel and state (16 per clock and SM) is the floor:
 * 119 us at 2 x 4096 x 4096 x 16, where the forward kernel takes 264 us: it waits, with two walking warps per scheduler and the
 * issue slots 48% busy, for shared memory, for arithmetic and at the barrier of each tile.  Backward, with dy the gradient of y:
 *   dh_t = C_t dy_t + a_{t+1} dh_{t+1},  a = exp(delta A);   da_t = dh_t h_{t-1} a_t (by the exponent)
 *   dA = sum of da delta,  ddelta = sum_n (da A + dh B x),  dx = delta sum_n dh B + D dy,
 *   dB = sum over channels of dh delta x,  dC = sum over channels of dy h,  dD = sum of dy x.
 */
#include <cfloat>

#include "seq_common.cuh"

namespace rpb_scan {

using namespace rpb_seq;

constexpr int NT = 128;             /* threads per block */
constexpr int S = 4;                /* states per thread */
constexpr int SEG = 8;              /* rows between two saved states: one backward segment, whose history is in registers */
constexpr int MAX_STATES = 64;

struct Args {
    int batch, len, channels, states, groups, softplus;
    long long x_batch, x_row, dt_batch, dt_row, b_batch, b_row, c_batch, c_row, z_batch, z_row, y_batch, y_row;
    long long dx_batch, dx_row, ddt_batch, ddt_row, dz_batch, dz_row;
    int per_group;                  /* channels of a group */
    int blocks;                     /* channel blocks of a group */
    int chunk, chunks;              /* rows per chunk (a multiple of the tile), and chunks per sequence */
    bool vec_x, vec_dt, vec_z, vec_y, vec_dx, vec_ddt, vec_dz, vec_n;
    bool fast;                      /* all operands that the call has, B and C among them, in whole packs */
};

/* P lanes per channel (4 states each), CH channels per block of NT walkers, tiles of TT rows; NL threads load a tile, V
 * channels of one row each. */
template <typename T, int P, int NL> struct Tile {
    static constexpr int CH = NT / P, TT = sizeof(T) >= 4 && P >= 4 ? 16 : P <= 4 ? 8 * P : 32, V = CH * TT / NL, NP = S * P;
    static constexpr int PAD = 32 / P;          /* rows of a [TT][CH] result are this much longer: P rows of a warp in 32 banks */
};

template <typename A> struct Pair { A delta, dx; };

/* The hardware's base-2 exponential is low on average: by 0.5e-8 to 2.5e-8 of its value for arguments from -1e-4 to -0.3
 * (2^20 each), and a state that decays slowly collects that over its whole memory: dA over 2 x 2048 rows was 9e-7 low on
 * average.  This much more in the exponent, in the multiply-add that forms it, leaves 9e-8 (3.6e-8 overshoots to +2.8e-7);
 * 2^CENTRE itself still is 1, so a delta of 0 changes nothing.  It is added to every exponent; those beyond -0.3, behind which little
 * of a state is left, were not measured one by one. */
constexpr float CENTRE = 2.5e-8f;
__device__ __forceinline__ float decay(float delta, float a) { return ex2_fast(fmaf(delta, a, CENTRE)); }
__device__ __forceinline__ double decay(double delta, double a) { return exp(delta * a); }
/* A as the decay wants it: in float times log2(e), for the base-2 exponential; finite, so that a delta of 0 (a row that is not part of
 * the sequence) changes nothing whatever A is */
__device__ __forceinline__ float decay_rate(float a) {
    float r;        /* NaN stays NaN */
    asm("{ .reg .f32 t; max.NaN.f32 t, %1, %2; min.NaN.f32 %0, t, %3; }" : "=f"(r) : "f"(a * 1.44269504088896341f), "f"(-FLT_MAX), "f"(FLT_MAX));
    return r;
}
__device__ __forceinline__ double decay_rate(double a) { return isinf(a) ? copysign(DBL_MAX, a) : a; }

__device__ __forceinline__ int row_end(const int* lengths, int b, int len) {
    if (!lengths) return len;
    const int n = lengths[b];
    return n < 0 ? 0 : n > len ? len : n;
}

/* four states from (to) a packed [.., states] row, 0 behind the last one */
template <typename A> __device__ __forceinline__ void load_states(A (&v)[S], const A* p, int n0, int states, bool vec) {
    const Pack<A, S> r = load_pack<A, S>(p + n0, states - n0, vec);
#pragma unroll
    for (int i = 0; i < S; ++i) v[i] = r.v[i];
}
template <typename A> __device__ __forceinline__ void store_states(A* p, const A (&v)[S], int n0, int states, bool vec) {
    Pack<A, S> r;
#pragma unroll
    for (int i = 0; i < S; ++i) r.v[i] = v[i];
    store_pack<A, S>(p + n0, r, states - n0, vec);
}

/* Sums v[0 .. G-1] over the M lanes whose numbers differ in the bits of M * UNIT - UNIT; lane m of them keeps the sums of
 * the G / M entries from m * (G / M) on (at least one: for G < M neighbouring lanes hold the same), in v[0 ..]. */
template <int G, int M, int UNIT, typename A> __device__ __forceinline__ void sum_lanes(A (&v)[G], int lane) {
    int left = G;
#pragma unroll
    for (int m = M / 2; m >= 1; m /= 2) {
        if (left > 1) {
            const int half = left / 2;
            const bool upper = lane & (m * UNIT);
#pragma unroll
            for (int i = 0; i < G / 2; ++i) {
                if (i >= half) continue;
                const A give = upper ? v[i] : v[i + half], keep = upper ? v[i + half] : v[i];
                v[i] = keep + __shfl_xor_sync(0xffffffffu, give, m * UNIT);
            }
            left = half;
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], m * UNIT);
        }
    }
}

/* V values at p, which is aligned for them, when `on`, else zeros: asynchronously into shared memory */
template <typename T, int V> __device__ __forceinline__ void bring(Pack<T, V>* to, const T* p, bool on) {
    constexpr int BYTES = sizeof(T) * V, STEP = BYTES < 16 ? BYTES : 16;
#pragma unroll
    for (int i = 0; i < BYTES; i += STEP) async_copy<STEP>(reinterpret_cast<char*>(to) + i, reinterpret_cast<const char*>(p) + i, on);
}
/* the same into registers, value by value: nothing is assumed about alignment */
template <typename T, int V> __device__ __forceinline__ void pick(Pack<T, V>& to, const T* p, bool on, int valid) {
    to = zero_pack<T, V>();
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (on && i < valid) to.v[i] = p[i];
}

/* Where a block works: sequence, group, first channel, channels left in the group, chunk of rows. */
struct Place { int b, g, d0, valid, c; };
template <int CH> __device__ __forceinline__ Place place_of(const Args& a) {
    Place p;
    long long i = blockIdx.x;
    const int per_seq = a.groups * a.blocks;
    const long long sc = i / per_seq;
    const int gb = (int)(i - sc * per_seq);
    p.b = (int)(sc / a.chunks); p.c = (int)(sc - (long long)p.b * a.chunks);
    p.g = gb / a.blocks;
    const int first = (gb - p.g * a.blocks) * CH;
    p.d0 = p.g * a.per_group + first;
    p.valid = a.per_group - first;
    return p;
}

/* h across a chunk whose deltas add up to `sum` and that ends with `part` from zero.  The chunk's decay in two halves: it may be
 * beyond the type's range where its product with h is not, and a state of 0 stays 0 however fast states grow. */
template <typename A> __device__ __forceinline__ void cross_chunk(A (&h)[S], const A (&part)[S], const A (&rate)[S], A sum) {
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const A half = decay(sum * A(0.5), rate[i]);
        h[i] = h[i] == A(0) ? part[i] : h[i] * half * half + part[i];
    }
}

/* Four states of one channel and their step: h = exp(delta A) h + dx b, and c . h.  In float the four are two register pairs
 * (mul / fma.f32x2: 13 instructions instead of 20 beside the four exponentials, which bound the scan). */
template <typename A> struct Walk {
    typedef Pack<A, S> Four;
    A h[S], rate[S];
    __device__ __forceinline__ void set_rate(const A (&r)[S]) { for (int i = 0; i < S; ++i) rate[i] = r[i]; }
    __device__ __forceinline__ void set(const A (&v)[S]) { for (int i = 0; i < S; ++i) h[i] = v[i]; }
    __device__ __forceinline__ void get(A (&v)[S]) const { for (int i = 0; i < S; ++i) v[i] = h[i]; }
    __device__ __forceinline__ void clear(const bool (&real)[S]) { for (int i = 0; i < S; ++i) h[i] = real[i] ? h[i] : A(0); }
    __device__ __forceinline__ void decays(Four& e, A delta) const {
#pragma unroll
        for (int i = 0; i < S; ++i) e.v[i] = decay(delta, rate[i]);
    }
    __device__ __forceinline__ void step(const Four& e, A dx, const Four& b) {
#pragma unroll
        for (int i = 0; i < S; ++i) h[i] = e.v[i] * h[i] + dx * b.v[i];
    }
    __device__ __forceinline__ A dot(const Four& c) const {
        A o = h[0] * c.v[0];
#pragma unroll
        for (int i = 1; i < S; ++i) o += h[i] * c.v[i];
        return o;
    }
};
template <> struct Walk<float> {
    typedef ulonglong2 Four;
    f32x2 h0, h1, r0, r1;
    __device__ __forceinline__ void set_rate(const float (&r)[S]) { r0 = pack2(r[0], r[1]); r1 = pack2(r[2], r[3]); }
    __device__ __forceinline__ void set(const float (&v)[S]) { h0 = pack2(v[0], v[1]); h1 = pack2(v[2], v[3]); }
    __device__ __forceinline__ void get(float (&v)[S]) const { unpack2(h0, v[0], v[1]); unpack2(h1, v[2], v[3]); }
    __device__ __forceinline__ void clear(const bool (&real)[S]) {
        float v[S];
        get(v);
#pragma unroll
        for (int i = 0; i < S; ++i) v[i] = real[i] ? v[i] : 0.0f;
        set(v);
    }
    __device__ __forceinline__ void decays(Four& e, float delta) const {
        const f32x2 dl = pack2(delta, delta);
        float e0, e1, e2, e3;
        unpack2(fma2(dl, r0, pack2(CENTRE, CENTRE)), e0, e1);
        unpack2(fma2(dl, r1, pack2(CENTRE, CENTRE)), e2, e3);
        e.x = pack2(ex2_fast(e0), ex2_fast(e1));
        e.y = pack2(ex2_fast(e2), ex2_fast(e3));
    }
    __device__ __forceinline__ void step(const Four& e, float dx, const Four& b) {
        const f32x2 d2 = pack2(dx, dx);
        h0 = fma2(e.x, h0, mul2(d2, b.x));
        h1 = fma2(e.y, h1, mul2(d2, b.y));
    }
    __device__ __forceinline__ float dot(const Four& c) const {
        float lo, hi;
        unpack2(fma2(h0, c.x, mul2(h1, c.y)), lo, hi);
        return lo + hi;
    }
};

/* ------------------------------------------------------------------------------------------------ forward
 * The shared layouts: a row of pairs is 16 bytes longer than its channels, so that the rows a warp of loaders writes at once
 * lie in other banks; a row of the walkers' parts of y holds the P parts of V channels, 4 words of padding, and so on, so that
 * the loaders' 16-byte reads of eight such groups meet no bank twice. */
template <typename T, int P> struct Forward : Tile<T, P, NT> {
    typedef Tile<T, P, NT> Base;
    static constexpr int NL = NT, K = Base::CH / Base::V;
    static constexpr int ROW = Base::CH + 2;
    static constexpr int YG = Base::V * P < 4 ? 4 : Base::V * P + 4, YROW = K * YG;
    static constexpr int UNITS = (Base::TT * P + NL - 1) / NL;      /* groups of four values of B (C) that a loader brings */
};

/*
 * Half of a block's threads walk: P lanes per channel, four states each, one tile of rows after the other.  The other half
 * load: while tile i is walked they turn tile i + 1 into deltas and delta x in shared memory (and B and C into floats) and
 * finish tile i - 1 (skip, gate, rounding, whole packs to memory); one barrier per tile.
 * AGG: the first of two passes over a long sequence that is split into chunks.  It leaves, per chunk, the state that the
 * chunk would end with from zero and the sum of its deltas; exp(A sum) is the whole chunk's decay, so the state in front of
 * a chunk is folded from these, and the second pass (AGG = false) runs every chunk from its own.
 * PADS: some of the P lanes' states are behind the last one.  They are cleared after every row: their B and C are 0, but 0 times an
 * infinite delta x would make them NaN, and y with them. */
template <typename T> struct Resident { static constexpr int value = sizeof(T) <= 4 ? 2 : 1; };

template <typename T, int P> struct Ring { static constexpr int DEPTH = P == 16 || sizeof(T) == 8 ? 1 : sizeof(T) == 4 ? 2 : 3, SLOTS = DEPTH + 2; };

template <typename T, int P, bool AGG> struct ForwardShared {
    typedef typename AccOf<T>::type A;
    typedef Forward<T, P> Sh;
    static constexpr int SLOTS = Ring<T, P>::SLOTS, ONE = AGG ? 1 : Sh::TT, NL = Sh::NL;
    Pack<T, Sh::V> raw_x[SLOTS][NL], raw_dt[SLOTS][NL], raw_z[AGG ? 1 : SLOTS][AGG ? 1 : NL];
    Pack<T, S> raw_b[SLOTS][Sh::TT * P], raw_c[AGG ? 1 : SLOTS][AGG ? 1 : Sh::TT * P];
    alignas(16) Pair<A> pairs[2][Sh::TT][Sh::ROW];
    alignas(16) A Bs[2][Sh::TT][Sh::NP], Cs[2][ONE][Sh::NP], ys[2][ONE][Sh::YROW];
};

template <typename T, int P, bool AGG, bool PADS>
__global__ void __launch_bounds__(NT + Forward<T, P>::NL, Resident<T>::value)
forward_kernel(T* __restrict__ y, typename AccOf<T>::type* h_out, typename AccOf<T>::type* __restrict__ saved, typename AccOf<T>::type* __restrict__ chunk_h,
               typename AccOf<T>::type* __restrict__ chunk_s, const T* __restrict__ x, const T* __restrict__ dt, const typename AccOf<T>::type* __restrict__ Am,
               const T* __restrict__ Bm, const T* __restrict__ Cm, const typename AccOf<T>::type* __restrict__ Dv,
               const typename AccOf<T>::type* __restrict__ dt_bias, const T* __restrict__ z, const typename AccOf<T>::type* h_in,
               const int* __restrict__ lengths, Args a) {
    typedef typename AccOf<T>::type A;
    typedef Forward<T, P> Sh;
    constexpr int CH = Sh::CH, TT = Sh::TT, V = Sh::V, NP = Sh::NP, YROW = Sh::YROW, NL = Sh::NL, K = Sh::K;
    extern __shared__ __align__(16) unsigned char raw_shared[];
    ForwardShared<T, P, AGG>& sh = *reinterpret_cast<ForwardShared<T, P, AGG>*>(raw_shared);
    static_assert(sizeof(sh) <= 227 * 1024 / Resident<T>::value - 1024, "");
    rpb_pdl_trigger();
    rpb_pdl_wait();
    const Place pl = place_of<CH>(a);
    const int end = row_end(lengths, pl.b, a.len);
    const int first = pl.c * a.chunk, last = first + a.chunk < a.len ? first + a.chunk : a.len;
    const int tiles = (last - first + TT - 1) / TT;

    if (threadIdx.x < NT) {
        const int tid = threadIdx.x, p = tid % P, ch = tid / P, n0 = p * S;
        const bool on = ch < pl.valid;
        const long long d = pl.d0 + ch;
        A rate[S], h[S], sum = 0;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            rate[i] = on && n0 + i < a.states ? decay_rate(Am[d * a.states + n0 + i]) : A(0);
            h[i] = 0;
        }
        /* the last chunk's slot holds a copy of h_in, which h_out may overwrite while other chunks have yet to begin */
        if (on && (a.chunks == 1 || (AGG && pl.c == a.chunks - 1))) {
            if (h_in) load_states(h, h_in + (pl.b * (long long)a.channels + d) * a.states, n0, a.states, a.vec_n);
            if (AGG) store_states(chunk_h + ((pl.b * (long long)a.chunks + pl.c) * a.channels + d) * a.states, h, n0, a.states, a.vec_n);
        }
        if (AGG && pl.c == a.chunks - 1) return;
        if (!AGG && on && a.chunks > 1) {
            load_states(h, chunk_h + ((pl.b * (long long)a.chunks + a.chunks - 1) * a.channels + d) * a.states, n0, a.states, a.vec_n);
#pragma unroll 4
            for (int c = 0; c < pl.c; ++c) {
                const long long at = (pl.b * (long long)a.chunks + c) * a.channels + d;
                A part[S];
                load_states(part, chunk_h + at * a.states, n0, a.states, a.vec_n);
                cross_chunk(h, part, rate, chunk_s[at]);
            }
        }
        Walk<A> w;
        bool real[S];
#pragma unroll
        for (int i = 0; i < S; ++i) real[i] = n0 + i < a.states;
        w.set(h);
        w.set_rate(rate);
        A* keep = nullptr;
        if (!AGG && saved && on) keep = saved + ((pl.b * (long long)((a.len + SEG - 1) / SEG) + first / SEG) * a.channels + d) * a.states;
        __syncthreads();
        for (int tile = 0; tile < tiles; ++tile) {
            const int buf = tile & 1, left = last - first - tile * TT;
            const Pair<A>* pairs = &sh.pairs[buf][0][ch];
            const A *bs = &sh.Bs[buf][0][n0], *cs = &sh.Cs[buf][0][n0];
            A* ys = &sh.ys[buf][0][AGG ? 0 : ch / V * Sh::YG + ch % V * P + p];
            /* The decays of a row are computed one row ahead of h's step; results wait in registers, since a store to shared
             * memory would hold up the loads behind it. */
            constexpr int BLK = TT < 16 ? TT : 16;
            typedef typename Walk<A>::Four Four;
#pragma unroll 1
            for (int t = 0; t < TT; t += BLK) {
                A v[BLK];
                Four e[2], bv[2], cv[2];
                Pair<A> pr[3] = {};
                auto bring = [&](int k) {
                    bv[k & 1] = *reinterpret_cast<const Four*>(bs + (t + k) * NP);
                    if (!AGG) cv[k & 1] = *reinterpret_cast<const Four*>(cs + (t + k) * NP);
                    w.decays(e[k & 1], pr[k % 3].delta);
                };
                pr[0] = pairs[t * Sh::ROW];
                pr[1] = pairs[(t + 1) * Sh::ROW];
                bring(0);
#pragma unroll
                for (int k = 0; k < BLK; ++k) {
                    if (!AGG && k % SEG == 0 && keep && t + k < left) {
                        w.get(h);
                        store_states(keep, h, n0, a.states, a.vec_n);
                        keep += (long long)a.channels * a.states;
                    }
                    if (k + 2 < BLK) pr[(k + 2) % 3] = pairs[(t + k + 2) * Sh::ROW];
                    if (k + 1 < BLK) bring(k + 1);
                    w.step(e[k & 1], pr[k % 3].dx, bv[k & 1]);
                    if (PADS) w.clear(real);
                    if (AGG) sum += pr[k % 3].delta;
                    else v[k] = w.dot(cv[k & 1]);
                }
                if (!AGG) {
#pragma unroll
                    for (int k = 0; k < BLK; ++k) ys[(t + k) * YROW] = v[k];
                }
            }
            __syncthreads();
        }
        if (!on) return;
        w.get(h);
        if (AGG) {
            const long long at = (pl.b * (long long)a.chunks + pl.c) * a.channels + d;
            store_states(chunk_h + at * a.states, h, n0, a.states, a.vec_n);
            if (p == 0) chunk_s[at] = sum;
        } else if (h_out && pl.c == a.chunks - 1) {
            store_states(h_out + (pl.b * (long long)a.channels + d) * a.states, h, n0, a.states, a.vec_n);
        }
        return;
    }

    if (AGG && pl.c == a.chunks - 1) return;
    /* The raw rows wait in a ring of shared memory, where each thread meets only what it brought itself: DEPTH tiles are on
     * their way while one is staged.  FAST: whole packs everywhere, a full block of channels, states in whole groups of four:
     * asynchronous copies; else plain loads. */
    auto load = [&](auto fast) {
        constexpr bool FAST = decltype(fast)::value;
        constexpr int UNITS = Sh::UNITS, DEPTH = Ring<T, P>::DEPTH, SLOTS = Ring<T, P>::SLOTS;
        const int tid = (int)threadIdx.x - NT;
        const int lr = tid / K, lk = tid % K, lc = lk * V, lvalid = FAST ? V : pl.valid - lc;
        const T* xp = x + pl.b * a.x_batch + (long long)(first + lr) * a.x_row + pl.d0 + lc;
        const T* dp = dt + pl.b * a.dt_batch + (long long)(first + lr) * a.dt_row + pl.d0 + lc;
        const T* zp = z ? z + pl.b * a.z_batch + (long long)(first + lr) * a.z_row + pl.d0 + lc : nullptr;
        T* yp = y + pl.b * a.y_batch + (long long)(first + lr) * a.y_row + pl.d0 + lc;
        const T* bp = Bm + pl.b * a.b_batch + pl.g * a.states + first * a.b_row;
        const T* cp = Cm + pl.b * a.c_batch + pl.g * a.states + first * a.c_row;
        A bias[V], skip[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            bias[i] = dt_bias && i < lvalid ? dt_bias[pl.d0 + lc + i] : A(0);
            skip[i] = !AGG && Dv && i < lvalid ? Dv[pl.d0 + lc + i] : A(0);
        }
        const int rows = (end < last ? end : last) - first;
        int t2 = 0, slot2 = 0;                      /* of the next fetch: row from `first`, slot of the ring */
        /* without FAST a tile's values wait in registers until the next iteration, which puts them into their slot */
        Pack<T, V> hold_x, hold_dt, hold_z;
        Pack<T, S> hold_b[UNITS], hold_c[UNITS];
        int held = -1;
        auto fetch = [&]() {
            const bool row = t2 + lr < rows;
            if (FAST) {
                bring(&sh.raw_x[slot2][tid], xp, row);
                bring(&sh.raw_dt[slot2][tid], dp, row);
                if (!AGG && z) bring(&sh.raw_z[slot2][AGG ? 0 : tid], zp, row);
            } else {
                pick(hold_x, xp, row, lvalid);
                pick(hold_dt, dp, row, lvalid);
                if (!AGG && z) pick(hold_z, zp, row, lvalid);
                held = slot2;
            }
#pragma unroll
            for (int k = 0; k < UNITS; ++k) {
                const int e = tid + k * NL, r = e / P, n = (e % P) * S;
                if (e >= TT * P) break;
                const bool in = t2 + r < rows && n < a.states;
                if (FAST) {
                    bring(&sh.raw_b[slot2][e], bp + r * a.b_row + n, in);
                    if (!AGG) bring(&sh.raw_c[slot2][AGG ? 0 : e], cp + r * a.c_row + n, in);
                } else {
                    pick(hold_b[k], bp + r * a.b_row + n, in, a.states - n);
                    if (!AGG) pick(hold_c[k], cp + r * a.c_row + n, in, a.states - n);
                }
            }
            t2 += TT;
            slot2 = slot2 + 1 == SLOTS ? 0 : slot2 + 1;
            xp += TT * a.x_row; dp += TT * a.dt_row; bp += TT * a.b_row; cp += TT * a.c_row;
            if (zp) zp += TT * a.z_row;
        };
        auto settle = [&]() {
            if (FAST || held < 0) return;
            sh.raw_x[held][tid] = hold_x;
            sh.raw_dt[held][tid] = hold_dt;
            if (!AGG && z) sh.raw_z[AGG ? 0 : held][AGG ? 0 : tid] = hold_z;
#pragma unroll
            for (int k = 0; k < UNITS; ++k) {
                const int e = tid + k * NL;
                if (e >= TT * P) break;
                sh.raw_b[held][e] = hold_b[k];
                if (!AGG) sh.raw_c[AGG ? 0 : held][AGG ? 0 : e] = hold_c[k];
            }
            held = -1;
        };
        auto stage = [&](int tile, int slot) {
            const bool row = tile * TT + lr < rows;
            const Pack<T, V> xr = sh.raw_x[slot][tid], dr = sh.raw_dt[slot][tid];
            A dl[V];
#pragma unroll
            for (int i = 0; i < V; ++i) dl[i] = up(dr.v[i]) + bias[i];
            if (a.softplus) softplus_all(dl);
            Pack<A, 2 * V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!row || i >= lvalid) dl[i] = 0;
                o.v[2 * i] = dl[i];
                o.v[2 * i + 1] = dl[i] * up(xr.v[i]);
            }
            *reinterpret_cast<Pack<A, 2 * V>*>(&sh.pairs[tile & 1][lr][lc]) = o;
#pragma unroll
            for (int k = 0; k < UNITS; ++k) {
                const int e = tid + k * NL, r = e / P, n = (e % P) * S;
                if (e < TT * P) {
                    Pack<A, S> v;
                    const Pack<T, S> br = sh.raw_b[slot][e];
#pragma unroll
                    for (int i = 0; i < S; ++i) v.v[i] = up(br.v[i]);
                    *reinterpret_cast<Pack<A, S>*>(&sh.Bs[tile & 1][r][n]) = v;
                    if (!AGG) {
                        const Pack<T, S> cr = sh.raw_c[slot][AGG ? 0 : e];
#pragma unroll
                        for (int i = 0; i < S; ++i) v.v[i] = up(cr.v[i]);
                        *reinterpret_cast<Pack<A, S>*>(&sh.Cs[tile & 1][AGG ? 0 : r][n]) = v;
                    }
                }
            }
        };
        auto finish = [&](int tile, int slot) {
            const int t = tile * TT + lr;
            if (first + t >= last || lvalid <= 0) return;
            const A* from = &sh.ys[tile & 1][AGG ? 0 : lr][lk * Sh::YG];
            constexpr int PART = V * P < 4 ? V * P : 4;
            alignas(16) A part[V * P];
#pragma unroll
            for (int j = 0; j < V * P; j += PART) *reinterpret_cast<Pack<A, PART>*>(&part[j]) = *reinterpret_cast<const Pack<A, PART>*>(from + j);
            const Pack<T, V> xr = sh.raw_x[slot][tid], zr = z ? sh.raw_z[slot][AGG ? 0 : tid] : zero_pack<T, V>();
            Pack<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) {
#pragma unroll
                for (int m = P / 2; m >= 1; m /= 2)
#pragma unroll
                    for (int j = 0; j < m; ++j) part[i * P + j] += part[i * P + j + m];
                A r = part[i * P] + skip[i] * up(xr.v[i]);
                if (z) { const A g = up(zr.v[i]); r *= g * logistic(g); }
                o.v[i] = down<T>(t < rows ? r : A(0));
            }
            T* to = yp + (long long)tile * TT * a.y_row;
            if (FAST) *reinterpret_cast<Pack<T, V>*>(to) = o;
            else store_pack<T, V>(to, o, lvalid, a.vec_y);
        };
        auto next = [](int slot) { return slot + 1 == SLOTS ? 0 : slot + 1; };
#pragma unroll
        for (int k = 0; k <= DEPTH; ++k) {
            settle();
            if (k < tiles) fetch();
            async_commit();
        }
        settle();
        async_wait<DEPTH>();
        stage(0, 0);
        __syncthreads();
        int done = SLOTS - 1, ahead = 1 % SLOTS;    /* slots of tile - 1 and tile + 1 */
        for (int tile = 0; tile < tiles; ++tile) {
            async_wait<DEPTH - 1>();                /* tile + 1 is there */
            settle();
            if (tile + 1 < tiles) stage(tile + 1, ahead);
            if (!AGG && tile > 0) finish(tile - 1, done);
            if (tile + 1 + DEPTH < tiles) fetch();  /* into the slot of tile - 1 */
            async_commit();
            done = next(done); ahead = next(ahead);
            __syncthreads();
        }
        if (!AGG) finish(tiles - 1, done);
    };
    if (a.fast && pl.valid >= CH) load(std::true_type());
    else load(std::false_type());
}

/* One token per sequence: what moves is the state, once in and once out.  P lanes per channel as above; each thread takes
 * the same channel of R sequences, so that A is read once for them and R states are on their way together. */
template <typename T, int P, int R>
__global__ void __launch_bounds__(256) token_kernel(T* __restrict__ y, typename AccOf<T>::type* h_out, const T* __restrict__ x, const T* __restrict__ dt,
                                                    const typename AccOf<T>::type* __restrict__ Am, const T* __restrict__ Bm, const T* __restrict__ Cm,
                                                    const typename AccOf<T>::type* __restrict__ Dv, const typename AccOf<T>::type* __restrict__ dt_bias,
                                                    const T* __restrict__ z, const typename AccOf<T>::type* h_in, const int* __restrict__ lengths, Args a,
                                                    int channel_blocks) {
    typedef typename AccOf<T>::type A;
    rpb_pdl_trigger();
    rpb_pdl_wait();
    const int group = blockIdx.x / channel_blocks;
    const int ch = ((int)(blockIdx.x - group * channel_blocks) * (int)blockDim.x + (int)threadIdx.x) / P;
    const int p = threadIdx.x % P, n0 = p * S, b0 = group * R;
    const bool on = ch < a.channels;
    const long long d = on ? ch : 0;
    const int g = (int)(d / a.per_group);
    A rate[S], h[R][S], xv[R], dl[R], zv[R], bv[R][S], cv[R][S];
    bool live[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int b = b0 + r;
        const bool in = on && b < a.batch;
        live[r] = in && row_end(lengths, b, 1) > 0;
#pragma unroll
        for (int i = 0; i < S; ++i) h[r][i] = 0;
        if (in && h_in) load_states(h[r], h_in + (b * (long long)a.channels + d) * a.states, n0, a.states, a.vec_n);
        xv[r] = live[r] ? up(x[b * a.x_batch + d]) : A(0);
        dl[r] = live[r] ? up(dt[b * a.dt_batch + d]) : A(0);
        zv[r] = live[r] && z ? up(z[b * a.z_batch + d]) : A(0);
        const int left = live[r] ? a.states - n0 : 0;
        const Pack<T, S> bp = load_pack<T, S>(Bm + b * a.b_batch + g * a.states + n0, left, a.fast);
        const Pack<T, S> cp = load_pack<T, S>(Cm + b * a.c_batch + g * a.states + n0, left, a.fast);
#pragma unroll
        for (int i = 0; i < S; ++i) { bv[r][i] = up(bp.v[i]); cv[r][i] = up(cp.v[i]); }
    }
    load_states(rate, Am + d * a.states, n0, a.states, a.vec_n);
    const A bias = dt_bias ? dt_bias[d] : A(0), skip = Dv ? Dv[d] : A(0);
#pragma unroll
    for (int i = 0; i < S; ++i) rate[i] = decay_rate(rate[i]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int b = b0 + r;
        A o[1] = {0};
        if (live[r]) {
            const A v = dl[r] + bias, delta = a.softplus ? softplus_of(v) : v, dx = delta * xv[r];
#pragma unroll
            for (int i = 0; i < S; ++i) {
                h[r][i] = decay(delta, rate[i]) * h[r][i] + dx * bv[r][i];
                if (n0 + i < a.states) o[0] += h[r][i] * cv[r][i];     /* not 0 times the NaN of an infinite dx times 0 */
            }
        }
        if (on && b < a.batch && h_out) store_states(h_out + (b * (long long)a.channels + d) * a.states, h[r], n0, a.states, a.vec_n);
        sum_lanes<1, P, 1>(o, threadIdx.x & 31);
        if (p == 0 && on && b < a.batch) {
            A out = o[0] + skip * xv[r];
            if (z) out *= zv[r] * logistic(zv[r]);
            y[b * a.y_batch + d] = down<T>(live[r] ? out : A(0));
        }
    }
}

/* Four states' worth of values: in float two register pairs, so that one instruction works on two. */
template <typename A> struct V4 {
    A v[S];
    __device__ __forceinline__ void set(const A (&x)[S]) { for (int i = 0; i < S; ++i) v[i] = x[i]; }
    __device__ __forceinline__ void get(A (&x)[S]) const { for (int i = 0; i < S; ++i) x[i] = v[i]; }
};
template <> struct V4<float> {
    f32x2 a, b;
    __device__ __forceinline__ void set(const float (&x)[S]) { a = pack2(x[0], x[1]); b = pack2(x[2], x[3]); }
    __device__ __forceinline__ void get(float (&x)[S]) const { unpack2(a, x[0], x[1]); unpack2(b, x[2], x[3]); }
};
template <typename A> __device__ __forceinline__ void clear(V4<A>& x, const bool (&real)[S]) {
    A v[S];
    x.get(v);
#pragma unroll
    for (int i = 0; i < S; ++i) v[i] = real[i] ? v[i] : A(0);
    x.set(v);
}
__device__ __forceinline__ V4<float> mul(const V4<float>& x, const V4<float>& y) { return {mul2(x.a, y.a), mul2(x.b, y.b)}; }
__device__ __forceinline__ V4<float> mul(const V4<float>& x, float y) { const f32x2 s = pack2(y, y); return {mul2(x.a, s), mul2(x.b, s)}; }
/* zeros formed from x: constants for them cost registers throughout the walk (594 us instead of 590 at 2 x 2048 x 4096 x 16); an
 * infinite x times 0 is NaN, and the larger of NaN and 0 is 0 */
__device__ __forceinline__ V4<float> zeros_like(const V4<float>& x) {
    float v[S];
    mul(x, 0.0f).get(v);
#pragma unroll
    for (int i = 0; i < S; ++i) v[i] = fmaxf(v[i], 0.0f);
    V4<float> r;
    r.set(v);
    return r;
}
__device__ __forceinline__ V4<double> zeros_like(const V4<double>&) { return {{0, 0, 0, 0}}; }
__device__ __forceinline__ V4<float> mad(const V4<float>& x, const V4<float>& y, const V4<float>& z) { return {fma2(x.a, y.a, z.a), fma2(x.b, y.b, z.b)}; }
__device__ __forceinline__ V4<float> mad(const V4<float>& x, float y, const V4<float>& z) { const f32x2 s = pack2(y, y); return {fma2(x.a, s, z.a), fma2(x.b, s, z.b)}; }
__device__ __forceinline__ float dot(const V4<float>& x, const V4<float>& y) {
    float lo, hi;
    unpack2(fma2(x.a, y.a, mul2(x.b, y.b)), lo, hi);
    return lo + hi;
}
__device__ __forceinline__ V4<float> decays(float delta, const V4<float>& rate) {
    float e0, e1, e2, e3;
    const f32x2 c = pack2(CENTRE, CENTRE);
    const V4<float> e = mad(rate, delta, {c, c});
    unpack2(e.a, e0, e1); unpack2(e.b, e2, e3);
    return {pack2(ex2_fast(e0), ex2_fast(e1)), pack2(ex2_fast(e2), ex2_fast(e3))};
}
/* (x0, x1, x2, x3) -> (x2, x3, x0, x1) */
__device__ __forceinline__ V4<float> swap_halves(const V4<float>& x, bool on) { return on ? V4<float>{x.b, x.a} : x; }
/* gives the upper half to lane ^ mask and adds what comes to the lower half */
__device__ __forceinline__ void fold_halves(const V4<float>& x, int mask, float& lo, float& hi) {
    float g0, g1;
    unpack2(x.b, g0, g1);
    g0 = __shfl_xor_sync(0xffffffffu, g0, mask); g1 = __shfl_xor_sync(0xffffffffu, g1, mask);
    unpack2(add2(x.a, pack2(g0, g1)), lo, hi);
}
__device__ __forceinline__ V4<double> mul(const V4<double>& x, const V4<double>& y) { V4<double> r; for (int i = 0; i < S; ++i) r.v[i] = x.v[i] * y.v[i]; return r; }
__device__ __forceinline__ V4<double> mul(const V4<double>& x, double y) { V4<double> r; for (int i = 0; i < S; ++i) r.v[i] = x.v[i] * y; return r; }
__device__ __forceinline__ V4<double> mad(const V4<double>& x, const V4<double>& y, const V4<double>& z) {
    V4<double> r; for (int i = 0; i < S; ++i) r.v[i] = x.v[i] * y.v[i] + z.v[i]; return r;
}
__device__ __forceinline__ V4<double> mad(const V4<double>& x, double y, const V4<double>& z) { V4<double> r; for (int i = 0; i < S; ++i) r.v[i] = x.v[i] * y + z.v[i]; return r; }
__device__ __forceinline__ double dot(const V4<double>& x, const V4<double>& y) { double r = x.v[0] * y.v[0]; for (int i = 1; i < S; ++i) r += x.v[i] * y.v[i]; return r; }
__device__ __forceinline__ V4<double> decays(double delta, const V4<double>& rate) { V4<double> r; for (int i = 0; i < S; ++i) r.v[i] = decay(delta, rate.v[i]); return r; }
__device__ __forceinline__ V4<double> swap_halves(const V4<double>& x, bool on) {
    V4<double> r; for (int i = 0; i < S; ++i) r.v[i] = on ? x.v[i ^ 2] : x.v[i]; return r;
}
__device__ __forceinline__ void fold_halves(const V4<double>& x, int mask, double& lo, double& hi) {
    lo = x.v[0] + __shfl_xor_sync(0xffffffffu, x.v[2], mask); hi = x.v[1] + __shfl_xor_sync(0xffffffffu, x.v[3], mask);
}

/* ------------------------------------------------------------------------------------------------ backward
 * Walkers and loaders as in the forward call, over a chunk's tiles from the last to the first.  Walkers take a tile in
 * segments of SEG rows: from the saved state in front of the segment they run the rows forward once more, with the states and
 * decays of all rows in registers, and then backward.  Sums over the states of a channel (for dx, ddt, dz) and over the
 * channels of a warp (for dB, dC) are taken by exchanging halves between lanes, so that every lane ends with a sum of its own.
 * Lanes of odd channels hold their four states with the halves swapped (from copies of B and C in that order): the half to
 * give away is then in the same registers in every lane, and the first and largest exchange needs no selection.
 * PADS: as in the forward call, for the states and their gradients; those of channels behind a group's last one too, whose zeros
 * would be multiplied by an infinite B or C on the way into dB and dC.
 * AGG: as in the forward call, from the chunk's end: the gradient that leaves the chunk's first row when none enters at its
 * end, and the sum of the deltas.
 * About 28 instructions per row, channel and state are 209 us of issue at 2 x 2048 x 4096 x 16, where it takes 410 us (1100 us before
 * loaders and walkers were apart and the exchanges without selections): the issue slots are 57% busy, and what the two walking
 * warps per scheduler wait for is arithmetic, shared memory and the barrier of each tile, in that order. */
template <typename T, int P> struct Backward {
    static constexpr int CH = NT / P, TT = P == 1 || sizeof(T) == 8 ? 8 : 16, NP = S * P, NL = NT;
    static constexpr int V = CH * TT >= NL ? CH * TT / NL : 1, K = CH / V;      /* loaders behind the TT-th row have nothing to do */
    static constexpr int ROW = CH + 2, QROW = CH + 4;
    static constexpr int UNITS = (TT * P + NL - 1) / NL;
    static constexpr int DEPTH = sizeof(T) == 2 ? 3 : sizeof(T) == 4 ? 2 : 1, SLOTS = DEPTH + 2;
    /* Blocks per SM that the registers allow, and whether walkers and loaders divide them unevenly: with up to 8 states both
     * have more to hold, and one block takes all. */
    static constexpr int RESIDENT = P <= 2 || sizeof(T) == 8 ? 1 : 2;
    static constexpr bool UNEVEN = RESIDENT == 2;
    static constexpr bool PACKS = sizeof(T) * V >= 4 && sizeof(T) * S >= 4;      /* large enough for asynchronous copies */
};

template <typename T, int P, bool AGG> struct BackwardShared {
    typedef typename AccOf<T>::type A;
    typedef Backward<T, P> Sh;
    static constexpr int SLOTS = Sh::SLOTS, NL = Sh::NL, TT = Sh::TT, ONE = AGG ? 1 : TT;
    Pack<T, Sh::V> raw_x[SLOTS][NL], raw_dt[SLOTS][NL], raw_z[SLOTS][NL], raw_dy[SLOTS][NL];
    Pack<T, S> raw_b[AGG ? 1 : SLOTS][AGG ? 1 : TT * P], raw_c[SLOTS][TT * P];
    alignas(16) Pair<A> pairs[2][TT][Sh::ROW];
    alignas(16) A dys[2][TT][Sh::QROW];
    alignas(16) A Bs[2][ONE][2][Sh::NP], Cs[2][TT][2][Sh::NP];
    alignas(16) A q[2][ONE][Sh::QROW], r[2][ONE][Sh::QROW], yc[2][ONE][Sh::QROW];
    alignas(16) A dB[2][NT / 32][ONE][Sh::NP], dC[2][NT / 32][ONE][Sh::NP];
};

template <typename T> struct Grads {
    typedef typename AccOf<T>::type A;
    T *dx, *ddt, *dz;
    A *dh_in, *parts, *part_b, *part_c;     /* parts: per (sequence, chunk) dA [channels, states], dD, ddt_bias [channels] */
    int acc_dx, acc_ddt, acc_dz;
    bool vec_part;                          /* part_b, part_c in whole groups of four */
};

/* 256 threads launched with 128 registers each: the walkers, who keep a segment's history, take 168 and the loaders 88 (the
 * launch makes sure of the 128: with fewer the walkers would wait for good) */
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <typename T, int P, bool AGG, bool PADS>
__global__ void __launch_bounds__(2 * NT, Backward<T, P>::RESIDENT)
backward_kernel(Grads<T> out, typename AccOf<T>::type* __restrict__ chunk_g, typename AccOf<T>::type* __restrict__ chunk_s, const T* __restrict__ dy,
                const typename AccOf<T>::type* __restrict__ dh_out, const T* __restrict__ x, const T* __restrict__ dt,
                const typename AccOf<T>::type* __restrict__ Am, const T* __restrict__ Bm, const T* __restrict__ Cm,
                const typename AccOf<T>::type* __restrict__ Dv, const typename AccOf<T>::type* __restrict__ dt_bias, const T* __restrict__ z,
                const int* __restrict__ lengths, const typename AccOf<T>::type* __restrict__ saved, Args a) {
    typedef typename AccOf<T>::type A;
    typedef Backward<T, P> Sh;
    constexpr int CH = Sh::CH, TT = Sh::TT, V = Sh::V, NP = Sh::NP, K = Sh::K, NL = Sh::NL;
    constexpr bool SPLIT = !AGG && Sh::UNEVEN;
    extern __shared__ __align__(16) unsigned char raw_shared[];
    BackwardShared<T, P, AGG>& sh = *reinterpret_cast<BackwardShared<T, P, AGG>*>(raw_shared);
    static_assert(sizeof(sh) <= 226 * 1024, "");
    rpb_pdl_trigger();
    rpb_pdl_wait();
    const Place pl = place_of<CH>(a);
    if (AGG && pl.c == 0) return;       /* nothing is in front of it */
    const int end = row_end(lengths, pl.b, a.len);
    const int first = pl.c * a.chunk, last = first + a.chunk < a.len ? first + a.chunk : a.len;
    const int rows = (end < last ? end : last) - first;         /* of the sequence, in this chunk; may be negative */
    const int tiles = (last - first + TT - 1) / TT;
    const long long D = a.channels;

    if (threadIdx.x < NT) {
        if (SPLIT) more_registers<168>();
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
        const int p = tid % P, ch = tid / P, n0 = p * S;
        const int odd = (lane / P) & 1;
        const bool on = ch < pl.valid;
        const long long d = pl.d0 + ch;
        V4<A> rate, Av, g, dA;
        A sum = 0;
        bool real[S];               /* PADS: the channel's states, in this lane's order */
#pragma unroll
        for (int i = 0; i < S; ++i) real[i] = on && n0 + (odd ? i ^ 2 : i) < a.states;
        {
            A t0[S], t1[S], z0[S];
#pragma unroll
            for (int i = 0; i < S; ++i) {
                t0[i] = on && n0 + i < a.states ? Am[d * a.states + n0 + i] : A(0);
                t1[i] = decay_rate(t0[i]);
                z0[i] = 0;
            }
            Av.set(t0); rate.set(t1); dA.set(z0);
            if (!AGG && on) {
                if (dh_out) load_states(z0, dh_out + (pl.b * D + d) * a.states, n0, a.states, a.vec_n);
#pragma unroll 4
                for (int c = a.chunks - 1; c > pl.c; --c) {
                    const long long at = (pl.b * (long long)a.chunks + c) * D + d;
                    load_states(t0, chunk_g + at * a.states, n0, a.states, a.vec_n);
                    cross_chunk(z0, t0, t1, chunk_s[at]);
                }
            }
            g.set(z0);
            Av = swap_halves(Av, odd); rate = swap_halves(rate, odd); g = swap_halves(g, odd);
        }
        /* the states in front of the segments, the next one's on their way while one is worked on */
        const long long seg_stride = D * a.states;
        const A* keep = nullptr;
        A h_next[S] = {0, 0, 0, 0};
        auto ahead = [&](int t) {           /* of the segment that begins at row t from `first` */
            if (keep && t >= 0 && first + t < last) load_states(h_next, keep + t / SEG * seg_stride, n0, a.states, a.vec_n);
        };
        if (!AGG && on) keep = saved + ((pl.b * (long long)((a.len + SEG - 1) / SEG) + first / SEG) * D + d) * a.states;
        if (!AGG) ahead(tiles * TT - SEG);
        __syncthreads();
        for (int it = 0; it < tiles; ++it) {
            const int buf = it & 1, t0 = (tiles - 1 - it) * TT;
            const Pair<A>* pairs = &sh.pairs[buf][0][ch];
            const A* dys = &sh.dys[buf][0][ch];
            const A *bs = &sh.Bs[buf][0][AGG ? 0 : odd][n0], *cs = &sh.Cs[buf][0][odd][n0];
            if constexpr (AGG) {
#pragma unroll 4
                for (int k = TT - 1; k >= 0; --k) {
                    const A dl = pairs[k * Sh::ROW].delta;
                    const V4<A> cv = *reinterpret_cast<const V4<A>*>(cs + k * 2 * NP);
                    sum += dl;
                    g = mul(mad(cv, dys[k * Sh::QROW], g), decays(dl, rate));
                }
            } else {
                /* dA of one tile, then added to the total: sums of at most 16 and of as many as there are tiles, where one sum
                 * over all rows would have lost a digit */
                V4<A> dA_tile = zeros_like(dA);
                /* PARTIAL: rows from `live` on are not part of the sequence (or the chunk).  Their decay is 1 and nothing enters,
                 * so the state and its gradient pass through them, and their results are 0 whatever the state holds. */
                auto segment = [&](int r0, int live, auto partial) {
                    constexpr bool PARTIAL = decltype(partial)::value;
                    V4<A> h0, av[SEG], h[SEG];
                    h0.set(h_next);
                    h0 = swap_halves(h0, odd);
                    ahead(t0 + r0 - SEG);
                    A yv[SEG], qv[SEG], rv[SEG];
#pragma unroll
                    for (int k = 0; k < SEG; ++k) {
                        const Pair<A> pr = pairs[(r0 + k) * Sh::ROW];
                        const V4<A> bv = *reinterpret_cast<const V4<A>*>(bs + (r0 + k) * 2 * NP);
                        const V4<A> cv = *reinterpret_cast<const V4<A>*>(cs + (r0 + k) * 2 * NP);
                        av[k] = decays(pr.delta, rate);
                        h[k] = mad(av[k], k ? h[k - 1] : h0, mul(bv, pr.dx));
                        if (PADS) clear(h[k], real);
                        yv[k] = dot(h[k], cv);
                    }
                    /* M lanes of a warp hold the same states of M channels; MS rows give one sum (or two) per lane */
                    constexpr int M = 32 / P, MS = M / S < 1 ? 1 : M / S, LEFT = MS * S / M;
                    static_assert(SEG % MS == 0, "");
                    A bsum[MS * 2], csum[MS * 2];
#pragma unroll
                    for (int k = SEG - 1; k >= 0; --k) {
                        const Pair<A> pr = pairs[(r0 + k) * Sh::ROW];
                        const A gy = dys[(r0 + k) * Sh::QROW];
                        const V4<A> bv = *reinterpret_cast<const V4<A>*>(bs + (r0 + k) * 2 * NP);
                        const V4<A> cv = *reinterpret_cast<const V4<A>*>(cs + (r0 + k) * 2 * NP);
                        A *b2 = &bsum[k % MS * 2], *c2 = &csum[k % MS * 2];
                        if (PARTIAL && k >= live) {
                            qv[k] = rv[k] = yv[k] = b2[0] = b2[1] = c2[0] = c2[1] = 0;
                        } else {
                            V4<A> dh = mad(cv, gy, g);
                            if (PADS) clear(dh, real);
                            g = mul(dh, av[k]);
                            const V4<A> da = mul(g, k ? h[k - 1] : h0);
                            qv[k] = dot(dh, bv);
                            rv[k] = dot(da, Av);
                            dA_tile = mad(da, pr.delta, dA_tile);
                            fold_halves(mul(dh, pr.dx), P, b2[0], b2[1]);
                            fold_halves(mul(h[k], gy), P, c2[0], c2[1]);
                        }
                        if (k % MS == 0) {
                            sum_lanes<MS * 2, M / 2, 2 * P>(bsum, lane);
                            sum_lanes<MS * 2, M / 2, 2 * P>(csum, lane);
#pragma unroll
                            for (int e = 0; e < LEFT; ++e) {
                                const int at = lane / (2 * P) * LEFT + e, row = r0 + k + at / 2, n = n0 + 2 * odd + at % 2;
                                sh.dB[buf][warp][row][n] = bsum[e];
                                sh.dC[buf][warp][row][n] = csum[e];
                            }
                        }
                    }
                    /* over the P lanes of a channel: G rows at a time, each lane left with one */
                    constexpr int G = P < SEG ? P : SEG;
#pragma unroll
                    for (int k = 0; k < SEG; k += G) {
                        A v0[G], v1[G], v2[G];
#pragma unroll
                        for (int i = 0; i < G; ++i) { v0[i] = qv[k + i]; v1[i] = rv[k + i]; v2[i] = yv[k + i]; }
                        sum_lanes<G, P, 1>(v0, lane);
                        sum_lanes<G, P, 1>(v1, lane);
                        if (z) sum_lanes<G, P, 1>(v2, lane);
                        const int mine = r0 + k + p / (P / G);
                        if (p % (P / G) == 0) { sh.q[buf][mine][ch] = v0[0]; sh.r[buf][mine][ch] = v1[0]; if (z) sh.yc[buf][mine][ch] = v2[0]; }
                    }
                };
                const int stop = rows - t0;
#pragma unroll 1
                for (int r0 = TT - SEG; r0 >= 0; r0 -= SEG) {
                    if (r0 + SEG <= stop) segment(r0, SEG, std::false_type());
                    else segment(r0, stop - r0, std::true_type());
                }
                dA = mad(dA_tile, A(1), dA);
            }
            __syncthreads();
        }
        if (!on) return;
        A v[S];
        swap_halves(g, odd).get(v);
        if (AGG) {
            const long long at = (pl.b * (long long)a.chunks + pl.c) * D + d;
            store_states(chunk_g + at * a.states, v, n0, a.states, a.vec_n);
            if (p == 0) chunk_s[at] = sum;
            return;
        }
        if (out.dh_in && pl.c == 0) store_states(out.dh_in + (pl.b * D + d) * a.states, v, n0, a.states, a.vec_n);
        if (out.parts) {
            swap_halves(dA, odd).get(v);
            store_states(out.parts + (pl.b * (long long)a.chunks + pl.c) * D * (a.states + 2) + d * a.states, v, n0, a.states, false);
        }
        return;
    }

    if (SPLIT) fewer_registers<88>();
    auto load = [&](auto fast) {
        constexpr bool FAST = decltype(fast)::value;
        constexpr int UNITS = Sh::UNITS, DEPTH = Sh::DEPTH, SLOTS = Sh::SLOTS;
        const int tid = (int)threadIdx.x - NT;
        const int lr = tid / K, lk = tid % K, lc = lk * V, lvalid = FAST ? V : pl.valid - lc;
        const bool busy = lr < TT;
        const int top = first + (tiles - 1) * TT;           /* first row of the tile that comes first */
        const T* xp = x + pl.b * a.x_batch + (long long)(top + lr) * a.x_row + pl.d0 + lc;
        const T* dp = dt + pl.b * a.dt_batch + (long long)(top + lr) * a.dt_row + pl.d0 + lc;
        const T* zp = z ? z + pl.b * a.z_batch + (long long)(top + lr) * a.z_row + pl.d0 + lc : nullptr;
        const T* gp = dy + pl.b * a.y_batch + (long long)(top + lr) * a.y_row + pl.d0 + lc;
        const T* bp = Bm + pl.b * a.b_batch + pl.g * a.states + top * a.b_row;
        const T* cp = Cm + pl.b * a.c_batch + pl.g * a.states + top * a.c_row;
        A bias[V], skip[V], gD[V], gbias[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            bias[i] = dt_bias && i < lvalid ? dt_bias[pl.d0 + lc + i] : A(0);
            skip[i] = !AGG && Dv && i < lvalid ? Dv[pl.d0 + lc + i] : A(0);
            gD[i] = gbias[i] = 0;
        }
        int t2 = (tiles - 1) * TT, slot2 = 0;       /* of the next fetch: row from `first`, slot of the ring */
        Pack<T, V> hold_x, hold_dt, hold_z, hold_dy;
        Pack<T, S> hold_b[UNITS], hold_c[UNITS];
        int held = -1;
        auto fetch = [&]() {
            const bool row = busy && t2 + lr < rows;
            if constexpr (FAST) {
                bring(&sh.raw_x[slot2][tid], xp, row);
                bring(&sh.raw_dt[slot2][tid], dp, row);
                if (z) bring(&sh.raw_z[slot2][tid], zp, row);
                bring(&sh.raw_dy[slot2][tid], gp, row);
            } else {
                pick(hold_x, xp, row, lvalid);
                pick(hold_dt, dp, row, lvalid);
                if (z) pick(hold_z, zp, row, lvalid);
                pick(hold_dy, gp, row, lvalid);
                held = slot2;
            }
#pragma unroll
            for (int k = 0; k < UNITS; ++k) {
                const int e = tid + k * NL, r = e / P, n = (e % P) * S;
                if (e >= TT * P) break;
                const bool in = t2 + r < rows && n < a.states;
                if constexpr (FAST) {
                    if (!AGG) bring(&sh.raw_b[AGG ? 0 : slot2][AGG ? 0 : e], bp + r * a.b_row + n, in);
                    bring(&sh.raw_c[slot2][e], cp + r * a.c_row + n, in);
                } else {
                    if (!AGG) pick(hold_b[k], bp + r * a.b_row + n, in, a.states - n);
                    pick(hold_c[k], cp + r * a.c_row + n, in, a.states - n);
                }
            }
            t2 -= TT;
            slot2 = slot2 + 1 == SLOTS ? 0 : slot2 + 1;
            xp -= TT * a.x_row; dp -= TT * a.dt_row; gp -= TT * a.y_row; bp -= TT * a.b_row; cp -= TT * a.c_row;
            if (zp) zp -= TT * a.z_row;
        };
        auto settle = [&]() {
            if (FAST || held < 0) return;
            sh.raw_x[held][tid] = hold_x;
            sh.raw_dt[held][tid] = hold_dt;
            if (z) sh.raw_z[held][tid] = hold_z;
            sh.raw_dy[held][tid] = hold_dy;
#pragma unroll
            for (int k = 0; k < UNITS; ++k) {
                const int e = tid + k * NL;
                if (e >= TT * P) break;
                if (!AGG) sh.raw_b[AGG ? 0 : held][AGG ? 0 : e] = hold_b[k];
                sh.raw_c[held][e] = hold_c[k];
            }
            held = -1;
        };
        auto copies = [&](A (*to)[NP], int n, const Pack<T, S>& from) {       /* both orders */
            Pack<A, S> v, w;
#pragma unroll
            for (int i = 0; i < S; ++i) { v.v[i] = up(from.v[i]); w.v[i ^ 2] = v.v[i]; }
            *reinterpret_cast<Pack<A, S>*>(&to[0][n]) = v;
            *reinterpret_cast<Pack<A, S>*>(&to[1][n]) = w;
        };
        auto stage = [&](int it, int slot) {
            const int buf = it & 1;
            if (busy) {
                const bool row = (tiles - 1 - it) * TT + lr < rows;
                const Pack<T, V> xr = sh.raw_x[slot][tid], dr = sh.raw_dt[slot][tid], gr = sh.raw_dy[slot][tid];
                const Pack<T, V> zr = z ? sh.raw_z[slot][tid] : zero_pack<T, V>();
                A dl[V];
#pragma unroll
                for (int i = 0; i < V; ++i) dl[i] = up(dr.v[i]) + bias[i];
                if (a.softplus) softplus_all(dl);
                Pack<A, 2 * V> o;
                Pack<A, V> gy;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (!row || i >= lvalid) dl[i] = 0;
                    o.v[2 * i] = dl[i];
                    o.v[2 * i + 1] = dl[i] * up(xr.v[i]);
                    A v = up(gr.v[i]);
                    if (z) { const A zv = up(zr.v[i]); v *= zv * logistic(zv); }
                    gy.v[i] = row && i < lvalid ? v : A(0);
                }
                *reinterpret_cast<Pack<A, 2 * V>*>(&sh.pairs[buf][lr][lc]) = o;
                *reinterpret_cast<Pack<A, V>*>(&sh.dys[buf][lr][lc]) = gy;
            }
#pragma unroll
            for (int k = 0; k < UNITS; ++k) {
                const int e = tid + k * NL, r = e / P, n = (e % P) * S;
                if (e >= TT * P) break;
                if (!AGG) copies(sh.Bs[buf][AGG ? 0 : r], n, sh.raw_b[AGG ? 0 : slot][AGG ? 0 : e]);
                copies(sh.Cs[buf][r], n, sh.raw_c[slot][e]);
            }
        };
        const long long all_rows = (long long)a.batch * a.len;
        const int blk = (pl.d0 - pl.g * a.per_group) / CH;
        auto finish = [&](int it, int slot) {
            const int buf = it & 1, t0 = (tiles - 1 - it) * TT;
            const long long t = first + t0 + lr;
            if (busy && t < last && lvalid > 0) {
                T* dxp = out.dx ? out.dx + pl.b * a.dx_batch + t * a.dx_row + pl.d0 + lc : nullptr;
                T* ddtp = out.ddt ? out.ddt + pl.b * a.ddt_batch + t * a.ddt_row + pl.d0 + lc : nullptr;
                T* dzp = out.dz ? out.dz + pl.b * a.dz_batch + t * a.dz_row + pl.d0 + lc : nullptr;
                Pack<T, V> o0 = zero_pack<T, V>(), o1 = o0, o2 = o0;
                if (dxp && out.acc_dx) o0 = load_pack<T, V>(dxp, lvalid, a.vec_dx);
                if (ddtp && out.acc_ddt) o1 = load_pack<T, V>(ddtp, lvalid, a.vec_ddt);
                if (dzp && out.acc_dz) o2 = load_pack<T, V>(dzp, lvalid, a.vec_dz);
                if (t0 + lr < rows) {
                    const Pack<T, V> xr = sh.raw_x[slot][tid], dr = sh.raw_dt[slot][tid], gr = sh.raw_dy[slot][tid];
                    const Pack<T, V> zr = z ? sh.raw_z[slot][tid] : zero_pack<T, V>();
                    const Pack<A, 2 * V> pr = *reinterpret_cast<const Pack<A, 2 * V>*>(&sh.pairs[buf][lr][lc]);
                    const Pack<A, V> gy = *reinterpret_cast<const Pack<A, V>*>(&sh.dys[buf][lr][lc]);
                    const Pack<A, V> q = *reinterpret_cast<const Pack<A, V>*>(&sh.q[buf][AGG ? 0 : lr][lc]);
                    const Pack<A, V> r = *reinterpret_cast<const Pack<A, V>*>(&sh.r[buf][AGG ? 0 : lr][lc]);
                    const Pack<A, V> yc = *reinterpret_cast<const Pack<A, V>*>(&sh.yc[buf][AGG ? 0 : lr][lc]);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        if (i >= lvalid) continue;
                        const A xv = up(xr.v[i]);
                        A dd = r.v[i] + xv * q.v[i];
                        if (a.softplus) dd *= logistic(up(dr.v[i]) + bias[i]);
                        o0.v[i] = down<T>(up(o0.v[i]) + pr.v[2 * i] * q.v[i] + skip[i] * gy.v[i]);
                        o1.v[i] = down<T>(up(o1.v[i]) + dd);
                        if (z) {
                            const A zv = up(zr.v[i]), s = logistic(zv);
                            o2.v[i] = down<T>(up(o2.v[i]) + up(gr.v[i]) * (yc.v[i] + skip[i] * xv) * s * (A(1) + zv * (A(1) - s)));
                        }
                        gD[i] += gy.v[i] * xv;
                        gbias[i] += dd;
                    }
                }
                if (dxp) store_pack<T, V>(dxp, o0, lvalid, a.vec_dx);
                if (ddtp) store_pack<T, V>(ddtp, o1, lvalid, a.vec_ddt);
                if (dzp) store_pack<T, V>(dzp, o2, lvalid, a.vec_dz);
            }
            /* the block's part of dB and dC: the warps' sums in turn */
            for (int e = tid; e < TT * P; e += NL) {
                const int r = e / P, n = (e % P) * S;
                if (first + t0 + r >= last || n >= a.states) continue;
                const long long at = ((blk * all_rows + (long long)pl.b * a.len + first + t0 + r) * a.groups + pl.g) * a.states + n;
#pragma unroll
                for (int which = 0; which < 2; ++which) {
                    A* to = which ? out.part_c : out.part_b;
                    if (!to) continue;
                    Pack<A, S> v = *reinterpret_cast<const Pack<A, S>*>(which ? &sh.dC[buf][0][AGG ? 0 : r][n] : &sh.dB[buf][0][AGG ? 0 : r][n]);
#pragma unroll
                    for (int w = 1; w < NT / 32; ++w) {
                        const Pack<A, S> u = *reinterpret_cast<const Pack<A, S>*>(which ? &sh.dC[buf][w][AGG ? 0 : r][n] : &sh.dB[buf][w][AGG ? 0 : r][n]);
#pragma unroll
                        for (int i = 0; i < S; ++i) v.v[i] += u.v[i];
                    }
                    store_pack<A, S>(to + at, v, a.states - n, out.vec_part);
                }
            }
        };
        auto next = [](int slot) { return slot + 1 == SLOTS ? 0 : slot + 1; };
#pragma unroll 1
        for (int k = 0; k <= DEPTH; ++k) {
            settle();
            if (k < tiles) fetch();
            async_commit();
        }
        settle();
        async_wait<DEPTH>();
        stage(0, 0);
        __syncthreads();
        int done = SLOTS - 1, next_slot = 1 % SLOTS;        /* slots of the tiles before and behind the one walked */
        for (int it = 0; it < tiles; ++it) {
            async_wait<DEPTH - 1>();                        /* tile it + 1 is there */
            settle();
            if (!AGG && it > 0) finish(it - 1, done);       /* before stage: it reads pairs and dys of the same buffer */
            if (it + 1 < tiles) stage(it + 1, next_slot);
            if (it + 1 + DEPTH < tiles) fetch();            /* into the slot of tile it - 1 */
            async_commit();
            done = next(done); next_slot = next(next_slot);
            __syncthreads();
        }
        if (AGG) return;
        finish(tiles - 1, done);
        if (!out.parts) return;
        /* the loaders' sums of one channel, a row of loaders after the other (in the memory of the pairs) */
        A* mine = &sh.pairs[0][0][0].delta;
        static_assert(sizeof(sh.pairs) >= sizeof(A) * 2 * NL * V, "");
        asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
        for (int i = 0; i < V; ++i) { mine[tid * V + i] = gD[i]; mine[NL * V + tid * V + i] = gbias[i]; }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        A* part = out.parts + (pl.b * (long long)a.chunks + pl.c) * D * (a.states + 2) + D * a.states;
        for (int c = tid; c < CH && c < pl.valid; c += NL) {
            A s0 = 0, s1 = 0;
            for (int r = 0; r < TT; ++r) {
                const int at = (r * K + c / V) * V + c % V;
                s0 += mine[at]; s1 += mine[NL * V + at];
            }
            part[pl.d0 + c] = s0;
            part[D + pl.d0 + c] = s1;
        }
    };
    if (Sh::PACKS && a.fast && pl.valid >= CH) load(std::integral_constant<bool, Sh::PACKS>());
    else load(std::false_type());
}

/* dB and dC (+)= the channel blocks' parts, [parts][rows][cols] -> rows of `cols` with the output's own strides */
template <typename T>
__global__ void __launch_bounds__(256) sum_blocks_kernel(T* __restrict__ out0, T* __restrict__ out1, const typename AccOf<T>::type* __restrict__ part0,
                                                         const typename AccOf<T>::type* __restrict__ part1, int n_parts, long long rows, int len, int cols,
                                                         long long batch0, long long row0, long long batch1, long long row1, int acc0, int acc1) {
    typedef typename AccOf<T>::type A;
    __shared__ A sums[8][33];
    rpb_pdl_trigger();
    rpb_pdl_wait();
    const bool second = blockIdx.y != 0;
    T* out = second ? out1 : out0;
    if (!out) return;
    const A* part = second ? part1 : part0;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const long long e = (long long)blockIdx.x * 32 + tx, total = rows * cols;
    A s = 0;
    if (e < total) {
#pragma unroll 8
        for (int i = ty; i < n_parts; i += 8) s += part[i * total + e];
    }
    sums[ty][tx] = s;
    __syncthreads();
    if (ty != 0 || e >= total) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) s += sums[i][tx];
    const long long r = e / cols, b = r / len, t = r - b * len;
    T* o = out + b * (second ? batch1 : batch0) + t * (second ? row1 : row0) + (e - r * cols);
    if (second ? acc1 : acc0) s += up(*o);
    *o = down<T>(s);
}

/* ------------------------------------------------------------------------------------------------ host */

int lanes_for(int states) {
    int p = 1;
    while (p * S < states) p *= 2;
    return p;
}

/* Rows per chunk.  Splitting a sequence costs a second pass over it (all of its exponentials again), so it pays only where
 * the channels alone leave most of the chip idle. */
int pick_chunk(const RpbScan* c) {
    const int ch = NT / lanes_for(c->states), tt = 32;      /* a multiple of every tile */
    const long long per_group = c->channels / c->groups;
    const long long warps = (long long)c->batch * c->groups * ((per_group + ch - 1) / ch) * (NT / 32);
    const int whole = (c->len + tt - 1) / tt * tt;
    if (warps >= SM_COUNT * 3 || c->len < 4 * tt) return whole;
    long long chunks = (SM_COUNT * 16 + warps - 1) / warps;
    if (chunks > 64) chunks = 64;
    long long chunk = (c->len + chunks - 1) / chunks;
    if (chunk < 2 * tt) chunk = 2 * tt;
    chunk = (chunk + tt - 1) / tt * tt;
    return chunk >= whole ? whole : (int)chunk;
}

const char* bad_geometry(const RpbScan* c, DType dtype) {
    if (!c) return "no geometry";
    if (!rpb_dtype_size((int)dtype)) return "unknown element type";
    if (c->batch <= 0 || c->len <= 0 || c->channels <= 0) return "batch, len and channels must be positive";
    if (c->batch > 1 << 30 || c->len > 1 << 30 || c->channels > 1 << 24) return "batch or len above 2^30, or channels above 2^24";
    if (c->states < 1 || c->states > MAX_STATES) return "states must be 1 to 64";
    if (c->groups < 1 || c->channels % c->groups != 0) return "groups must divide the channels";
    if (c->softplus != 0 && c->softplus != 1) return "softplus must be 0 or 1";
    return nullptr;
}

Args make_args(const RpbScan* c) {
    Args a;
    a.batch = c->batch; a.len = c->len; a.channels = c->channels; a.states = c->states; a.groups = c->groups; a.softplus = c->softplus;
    a.x_batch = c->x_batch; a.x_row = c->x_row; a.dt_batch = c->dt_batch; a.dt_row = c->dt_row;
    a.b_batch = c->b_batch; a.b_row = c->b_row; a.c_batch = c->c_batch; a.c_row = c->c_row;
    a.z_batch = c->z_batch; a.z_row = c->z_row; a.y_batch = c->y_batch; a.y_row = c->y_row;
    a.dx_batch = c->dx_batch; a.dx_row = c->dx_row; a.ddt_batch = c->ddt_batch; a.ddt_row = c->ddt_row;
    a.dz_batch = c->dz_batch; a.dz_row = c->dz_row;
    a.per_group = c->channels / c->groups;
    const int ch = NT / lanes_for(c->states);
    a.blocks = (a.per_group + ch - 1) / ch;
    a.chunk = pick_chunk(c);
    a.chunks = (c->len + a.chunk - 1) / a.chunk;
    a.vec_x = a.vec_dt = a.vec_z = a.vec_y = a.vec_dx = a.vec_ddt = a.vec_dz = a.vec_n = a.fast = false;
    return a;
}

struct Rowset { Rows x, dt, B, C, z, y; };
Rowset rows_of(const RpbScan* c, const void* x, const void* dt, const void* B, const void* C, const void* z, const void* y) {
    const long long gn = (long long)c->groups * c->states;
    return {{x, c->x_batch, c->x_row, c->channels}, {dt, c->dt_batch, c->dt_row, c->channels}, {B, c->b_batch, c->b_row, gn},
            {C, c->c_batch, c->c_row, gn}, {z, c->z_batch, c->z_row, c->channels}, {y, c->y_batch, c->y_row, c->channels}};
}

/* whole packs of V channels: the rows are aligned, and so is the first channel of every block */
template <typename T, int V> bool packs_ok(const RpbScan* c, const Rows& r) {
    const size_t bytes = sizeof(T) * V < 16 ? sizeof(T) * V : 16;
    return r.p && aligned_rows(r, c->batch, c->len, sizeof(T), bytes) && (c->groups == 1 || (c->channels / c->groups) % V == 0);
}
/* B and C in groups of four states */
template <typename T> bool quads_ok(const RpbScan* c, const Rows& r) {
    const size_t bytes = sizeof(T) * S < 16 ? sizeof(T) * S : 16;
    return c->states % S == 0 && aligned_rows(r, c->batch, c->len, sizeof(T), bytes);
}
template <typename A> bool states_ok(const RpbScan* c, const void* p) {
    return !p || (c->states % S == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0);
}

template <typename T>
long long chunk_bytes(const RpbScan* c) {
    const int chunk = pick_chunk(c);
    const long long chunks = (c->len + chunk - 1) / chunk;
    if (chunks == 1) return 0;
    return ((long long)c->batch * chunks * c->channels * (c->states + 1) + 3) / 4 * 4 * (long long)sizeof(typename AccOf<T>::type);
}

template <typename T>
long long grad_bytes(const RpbScan* c) {
    const long long es = sizeof(typename AccOf<T>::type), chunk = pick_chunk(c), chunks = (c->len + chunk - 1) / chunk;
    const int ch = NT / lanes_for(c->states);
    const long long blocks = (c->channels / c->groups + ch - 1) / ch;
    return chunk_bytes<T>(c) + es * ((long long)c->batch * chunks * c->channels * (c->states + 2) +
                                     2 * blocks * c->batch * c->len * c->groups * c->states);
}

struct Operands {
    const void *x, *dt, *A, *B, *C, *D, *dt_bias, *z;
    const int* lengths;
};

template <typename T, int P, bool PADS>
int forward_p(void* y, void* h_out, void* saved, const Operands& o, const void* h_in, void* ws, const RpbScan* c, cudaStream_t s) {
    typedef typename AccOf<T>::type A;
    typedef Forward<T, P> Sh;
    Args a = make_args(c);
    const Rowset r = rows_of(c, o.x, o.dt, o.B, o.C, o.z, y);
    const A *Am = reinterpret_cast<const A*>(o.A), *Dv = reinterpret_cast<const A*>(o.D), *bias = reinterpret_cast<const A*>(o.dt_bias);
    const T *x = reinterpret_cast<const T*>(o.x), *dt = reinterpret_cast<const T*>(o.dt), *B = reinterpret_cast<const T*>(o.B);
    const T *C = reinterpret_cast<const T*>(o.C), *z = reinterpret_cast<const T*>(o.z);
    const A* hi = reinterpret_cast<const A*>(h_in);
    A* ho = reinterpret_cast<A*>(h_out);
    a.vec_n = states_ok<A>(c, h_in) && states_ok<A>(c, h_out);
    if (c->len == 1 && !saved) {
        a.vec_n = a.vec_n && states_ok<A>(c, o.A);
        a.fast = quads_ok<T>(c, r.B) && quads_ok<T>(c, r.C);
        constexpr int R = 2, BLOCK = 128;      /* 12.2 us for 64 x 4096 x 16 (R = 1: 12.5, R = 4: 15.5) */
        const int channel_blocks = (c->channels * P + BLOCK - 1) / BLOCK;
        const long long blocks = (long long)((c->batch + R - 1) / R) * channel_blocks;
        if (blocks > 0x7fffffffLL) return refuse("rp_selective_scan_ex", "too many sequences for one launch");
        SEQ_CUDA(rpb_launch(token_kernel<T, P, R>, dim3((unsigned)blocks), dim3(BLOCK), 0, s, 1, reinterpret_cast<T*>(y), ho, x, dt, Am, B, C, Dv, bias, z,
                            hi, o.lengths, a, channel_blocks));
        rpb_count_launches(1);
        return 0;
    }
    a.vec_x = packs_ok<T, Sh::V>(c, r.x); a.vec_dt = packs_ok<T, Sh::V>(c, r.dt);
    a.vec_z = packs_ok<T, Sh::V>(c, r.z); a.vec_y = packs_ok<T, Sh::V>(c, r.y);
    a.vec_n = a.vec_n && states_ok<A>(c, saved) && states_ok<A>(c, ws);
    a.fast = a.vec_x && a.vec_dt && (!z || a.vec_z) && a.vec_y && quads_ok<T>(c, r.B) && quads_ok<T>(c, r.C);
    const long long blocks = (long long)c->batch * a.chunks * c->groups * a.blocks;
    if (blocks > 0x7fffffffLL) return refuse("rp_selective_scan_ex", "too many sequences for one launch");
    A* chunk_h = reinterpret_cast<A*>(ws);
    A* chunk_s = chunk_h ? chunk_h + (long long)c->batch * a.chunks * c->channels * c->states : nullptr;
    static unsigned char done[2][64];
    int device = 0;
    SEQ_CUDA(cudaGetDevice(&device));
    if (allow_shared(forward_kernel<T, P, true, false>, sizeof(ForwardShared<T, P, true>), device, done[0]) ||
        allow_shared(forward_kernel<T, P, false, PADS>, sizeof(ForwardShared<T, P, false>), device, done[1])) return -1;
    if (a.chunks > 1) {
        SEQ_CUDA(rpb_launch(forward_kernel<T, P, true, false>, dim3((unsigned)blocks), dim3(NT + Forward<T, P>::NL), sizeof(ForwardShared<T, P, true>), s, 1, reinterpret_cast<T*>(y), ho, reinterpret_cast<A*>(saved),
                            chunk_h, chunk_s, x, dt, Am, B, C, Dv, bias, z, hi, o.lengths, a));
        rpb_count_launches(1);
    }
    SEQ_CUDA(rpb_launch(forward_kernel<T, P, false, PADS>, dim3((unsigned)blocks), dim3(NT + Forward<T, P>::NL), sizeof(ForwardShared<T, P, false>), s, 1, reinterpret_cast<T*>(y), ho, reinterpret_cast<A*>(saved),
                        chunk_h, chunk_s, x, dt, Am, B, C, Dv, bias, z, hi, o.lengths, a));
    rpb_count_launches(1);
    return 0;
}

struct Wanted {
    void *dx, *ddt, *dA, *dB, *dC, *dD, *ddt_bias, *dz, *dh_in;
    int accumulate;
};

template <typename T, int P, bool PADS>
int backward_p(const Wanted& w, const void* dy, const void* dh_out, const Operands& o, const void* saved, void* ws, const RpbScan* c,
               cudaStream_t s) {
    typedef typename AccOf<T>::type A;
    typedef Backward<T, P> Sh;
    Args a = make_args(c);
    const Rowset r = rows_of(c, o.x, o.dt, o.B, o.C, o.z, dy);
    const A *Am = reinterpret_cast<const A*>(o.A), *Dv = reinterpret_cast<const A*>(o.D), *bias = reinterpret_cast<const A*>(o.dt_bias);
    const T *x = reinterpret_cast<const T*>(o.x), *dt = reinterpret_cast<const T*>(o.dt), *B = reinterpret_cast<const T*>(o.B);
    const T *C = reinterpret_cast<const T*>(o.C), *z = reinterpret_cast<const T*>(o.z), *g = reinterpret_cast<const T*>(dy);
    a.vec_x = packs_ok<T, Sh::V>(c, r.x); a.vec_dt = packs_ok<T, Sh::V>(c, r.dt);
    a.vec_z = packs_ok<T, Sh::V>(c, r.z); a.vec_y = packs_ok<T, Sh::V>(c, r.y);
    a.vec_dx = packs_ok<T, Sh::V>(c, {w.dx, c->dx_batch, c->dx_row, c->channels});
    a.vec_ddt = packs_ok<T, Sh::V>(c, {w.ddt, c->ddt_batch, c->ddt_row, c->channels});
    a.vec_dz = packs_ok<T, Sh::V>(c, {w.dz, c->dz_batch, c->dz_row, c->channels});
    a.vec_n = states_ok<A>(c, saved) && states_ok<A>(c, ws) && states_ok<A>(c, dh_out) && states_ok<A>(c, w.dh_in);
    const long long blocks = (long long)c->batch * a.chunks * c->groups * a.blocks;
    if (blocks > 0x7fffffffLL) return refuse("rp_selective_scan_grad_ex", "too many sequences for one launch");
    const long long rows = (long long)c->batch * c->len, cols = (long long)c->groups * c->states;
    A* chunk_g = reinterpret_cast<A*>(ws);
    A* chunk_s = chunk_g + (long long)c->batch * a.chunks * c->channels * c->states;
    A* parts = reinterpret_cast<A*>(reinterpret_cast<char*>(ws) + chunk_bytes<T>(c));
    A* part_b = parts + (long long)c->batch * a.chunks * c->channels * (c->states + 2);
    A* part_c = part_b + a.blocks * rows * cols;
    Grads<T> out;
    out.dx = reinterpret_cast<T*>(w.dx); out.ddt = reinterpret_cast<T*>(w.ddt); out.dz = reinterpret_cast<T*>(w.dz);
    out.dh_in = reinterpret_cast<A*>(w.dh_in);
    out.parts = w.dA || w.dD || w.ddt_bias ? parts : nullptr;
    out.part_b = w.dB ? part_b : nullptr; out.part_c = w.dC ? part_c : nullptr;
    out.acc_dx = (w.accumulate & RPB_SCAN_ACC_DX) != 0; out.acc_ddt = (w.accumulate & RPB_SCAN_ACC_DDT) != 0;
    out.acc_dz = (w.accumulate & RPB_SCAN_ACC_DZ) != 0;
    out.vec_part = c->states % S == 0 && reinterpret_cast<uintptr_t>(part_b) % 16 == 0 && reinterpret_cast<uintptr_t>(part_c) % 16 == 0;
    a.fast = a.vec_x && a.vec_dt && (!z || a.vec_z) && a.vec_y && quads_ok<T>(c, r.B) && quads_ok<T>(c, r.C);
    const size_t agg = sizeof(BackwardShared<T, P, true>), smem = sizeof(BackwardShared<T, P, false>);
    static unsigned char done[2][64];
    int device = 0;
    SEQ_CUDA(cudaGetDevice(&device));
    if (allow_shared(backward_kernel<T, P, true, false>, agg, device, done[0]) || allow_shared(backward_kernel<T, P, false, PADS>, smem, device, done[1])) return -1;
    if (Sh::UNEVEN) {
        static int registers = 0;       /* the same on every device */
        if (registers == 0) {
            cudaFuncAttributes attr;
            SEQ_CUDA(cudaFuncGetAttributes(&attr, backward_kernel<T, P, false, PADS>));
            registers = attr.numRegs;
        }
        if (registers != 128) return refuse("rp_selective_scan_grad_ex", "built with another number of registers than its kernel divides");
    }
    const A* dho = reinterpret_cast<const A*>(dh_out);
    const A* sv = reinterpret_cast<const A*>(saved);
    if (a.chunks > 1) {
        SEQ_CUDA(rpb_launch(backward_kernel<T, P, true, false>, dim3((unsigned)blocks), dim3(2 * NT), agg, s, 1, out, chunk_g, chunk_s, g, dho, x, dt, Am, B, C, Dv, bias,
                            z, o.lengths, sv, a));
        rpb_count_launches(1);
    }
    SEQ_CUDA(rpb_launch(backward_kernel<T, P, false, PADS>, dim3((unsigned)blocks), dim3(2 * NT), smem, s, 1, out, chunk_g, chunk_s, g, dho, x, dt, Am, B, C, Dv, bias, z,
                        o.lengths, sv, a));
    rpb_count_launches(1);
    if (w.dB || w.dC) {
        const long long sum_blocks = (rows * cols + 31) / 32;
        if (sum_blocks > 0x7fffffffLL) return refuse("rp_selective_scan_grad_ex", "too many rows for one launch");
        SEQ_CUDA(rpb_launch(sum_blocks_kernel<T>, dim3((unsigned)sum_blocks, 2), dim3(256), 0, s, 1, reinterpret_cast<T*>(w.dB), reinterpret_cast<T*>(w.dC),
                            (const A*)part_b, (const A*)part_c, a.blocks, rows, c->len, (int)cols, c->db_batch, c->db_row, c->dc_batch, c->dc_row,
                            (w.accumulate & RPB_SCAN_ACC_DB) != 0, (w.accumulate & RPB_SCAN_ACC_DC) != 0));
        rpb_count_launches(1);
    }
    if (!out.parts) return 0;
    const long long D = c->channels, N = c->states;
    PartSums d = {};
    d.out[0] = w.dA; d.first[0] = 0; d.cols[0] = D * N; d.accumulate[0] = (w.accumulate & RPB_SCAN_ACC_DA) != 0;
    d.out[1] = w.dD; d.first[1] = D * N; d.cols[1] = D; d.accumulate[1] = (w.accumulate & RPB_SCAN_ACC_DD) != 0;
    d.out[2] = w.ddt_bias; d.first[2] = D * (N + 1); d.cols[2] = D; d.accumulate[2] = (w.accumulate & RPB_SCAN_ACC_DDT_BIAS) != 0;
    return sum_parts<A>(d, parts, c->batch * a.chunks, D * (N + 2), s);
}

/* The lanes of a channel, and whether they have states behind the last one (or, where `per_group` is given, a group's last block
 * channels behind the last one). */
template <typename F> int by_lanes(int states, int per_group, F f) {
#define CASE(n)                                                                                              \
    case n:                                                                                                  \
        return states == n * S && per_group % (NT / n) == 0 ? f(std::integral_constant<int, n>(), std::false_type()) \
                                                            : f(std::integral_constant<int, n>(), std::true_type());
    switch (lanes_for(states)) { CASE(1) CASE(2) CASE(4) CASE(8) CASE(16) }
#undef CASE
    return -1;
}

template <typename F> int by_type(DType dtype, F f) {
    switch ((int)dtype) {
        case DTYPE_FLOAT32: return f(float());
        case DTYPE_FLOAT64: return f(double());
        case DTYPE_FLOAT16: return f(__half());
        case DTYPE_BFLOAT16: return f(__nv_bfloat16());
    }
    return -1;
}

/* what both directions check about the operands that they read */
const char* bad_operands(const RpbScan* c, const Rowset& r, const Operands& o, bool z_given) {
    if (!o.x || !o.dt || !o.A || !o.B || !o.C) return "x, dt, A, B and C are needed";
    if (!readable(r.x, c->batch, c->len)) return "strides of x";
    if (!readable(r.dt, c->batch, c->len)) return "strides of dt";
    if (!readable(r.B, c->batch, c->len)) return "strides of B";
    if (!readable(r.C, c->batch, c->len)) return "strides of C";
    if (z_given && !readable(r.z, c->batch, c->len)) return "strides of z";
    return nullptr;
}

}  // namespace rpb_scan

using namespace rpb_seq;
using namespace rpb_scan;

extern "C" {

void rpb_scan_packed(RpbScan* c, int batch, int len, int channels, int states, int groups, int softplus) {
    memset(c, 0, sizeof(*c));
    c->batch = batch; c->len = len; c->channels = channels; c->states = states; c->groups = groups; c->softplus = softplus;
    c->x_row = c->dt_row = c->z_row = c->y_row = c->dx_row = c->ddt_row = c->dz_row = channels;
    c->x_batch = c->dt_batch = c->z_batch = c->y_batch = c->dx_batch = c->ddt_batch = c->dz_batch = (long long)len * channels;
    c->b_row = c->c_row = c->db_row = c->dc_row = (long long)groups * states;
    c->b_batch = c->c_batch = c->db_batch = c->dc_batch = (long long)len * groups * states;
}

long long rp_selective_scan_saved_elems(const RpbScan* c, DType dtype) {
    const char* why = bad_geometry(c, dtype);
    if (why) return refuse("rp_selective_scan_saved_elems", why);
    return (long long)c->batch * ((c->len + SEG - 1) / SEG) * c->channels * c->states;
}

long long rp_selective_scan_ws_bytes(const RpbScan* c, DType dtype, int grad) {
    const char* why = bad_geometry(c, dtype);
    if (why) return refuse("rp_selective_scan_ws_bytes", why);
    if ((int)dtype == DTYPE_FLOAT64) return grad ? grad_bytes<double>(c) : chunk_bytes<double>(c);
    return grad ? grad_bytes<float>(c) : chunk_bytes<float>(c);
}

int rp_selective_scan_ex(void* y, void* h_out, void* saved, const void* x, const void* dt, const void* A, const void* B, const void* C, const void* D,
                         const void* dt_bias, const void* z, const void* h_in, const int* lengths, void* ws, const RpbScan* c, DType dtype,
                         int device_id, void* stream) {
    const char* name = "rp_selective_scan_ex";
    const char* why = bad_geometry(c, dtype);
    if (why) return refuse(name, why);
    if (!y) return refuse(name, "y is needed");
    if (device_id < 0) return refuse(name, "needs a CUDA device (no CPU path in this library)");
    const Operands o = {x, dt, A, B, C, D, dt_bias, z, lengths};
    const Rowset r = rows_of(c, x, dt, B, C, z, y);
    why = bad_operands(c, r, o, z != nullptr);
    if (why) return refuse(name, why);
    if (!writable(r.y, c->batch, c->len)) return refuse(name, "strides of y");
    const long long ws_bytes = rp_selective_scan_ws_bytes(c, dtype, 0), d = c->channels, all = (long long)c->batch * d * c->states;
    if (!ws && ws_bytes > 0) return refuse(name, "this size needs a workspace");
    const size_t es = rpb_dtype_size((int)dtype), as = dtype == DTYPE_FLOAT64 ? 8 : 4;
    auto area = [&](const char* n, const Rows& rows) { return strided(n, rows, c->batch, c->len, es); };
    const Area outs[] = {area("y", r.y), packed("h_out", h_out, all, as, h_in), packed("saved", saved, rp_selective_scan_saved_elems(c, dtype), as),
                         packed("ws", ws, ws_bytes / (long long)as, as)};
    const Area ins[] = {area("x", r.x), area("dt", r.dt), area("B", r.B), area("C", r.C), area("z", r.z), packed("A", A, d * c->states, as),
                        packed("D", D, d, as), packed("dt_bias", dt_bias, d, as), packed("h_in", h_in, all, as),
                        packed("lengths", lengths, c->batch, sizeof(int))};
    if (refuse_buffers(name, outs, ins)) return -1;
    DeviceScope scope;
    if (scope.enter(device_id)) return refuse(name, "no such device");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return by_type(dtype, [&](auto t) {
        return by_lanes(c->states, 0, [&](auto p, auto pads) { return forward_p<decltype(t), decltype(p)::value, decltype(pads)::value>(y, h_out, saved, o, h_in, ws, c, s); });
    });
}

int rp_selective_scan_grad_ex(void* dx, void* ddt, void* dA, void* dB, void* dC, void* dD, void* ddt_bias, void* dz, void* dh_in, int accumulate,
                              const void* dy, const void* dh_out, const void* x, const void* dt, const void* A, const void* B, const void* C,
                              const void* D, const void* dt_bias, const void* z, const int* lengths, const void* saved, void* ws, const RpbScan* c,
                              DType dtype, int device_id, void* stream) {
    const char* name = "rp_selective_scan_grad_ex";
    const char* why = bad_geometry(c, dtype);
    if (why) return refuse(name, why);
    if (!dx && !ddt && !dA && !dB && !dC && !dD && !ddt_bias && !dz && !dh_in) return refuse(name, "no gradient is wanted");
    if (!dy || !saved || !ws) return refuse(name, "dy, the saved states of the forward call and a workspace are needed");
    if (dz && !z) return refuse(name, "dz without z");
    if (device_id < 0) return refuse(name, "needs a CUDA device (no CPU path in this library)");
    const Operands o = {x, dt, A, B, C, D, dt_bias, z, lengths};
    const Rowset r = rows_of(c, x, dt, B, C, z, dy);
    why = bad_operands(c, r, o, z != nullptr);
    if (why) return refuse(name, why);
    if (!readable(r.y, c->batch, c->len)) return refuse(name, "strides of dy");
    const long long gn = (long long)c->groups * c->states;
    const Rows w[5] = {{dx, c->dx_batch, c->dx_row, c->channels}, {ddt, c->ddt_batch, c->ddt_row, c->channels}, {dz, c->dz_batch, c->dz_row, c->channels},
                       {dB, c->db_batch, c->db_row, gn}, {dC, c->dc_batch, c->dc_row, gn}};
    const size_t es = rpb_dtype_size((int)dtype);
    for (const Rows& g : w)
        if (g.p && !writable(g, c->batch, c->len)) return refuse(name, "strides of a gradient");
    const size_t as = dtype == DTYPE_FLOAT64 ? 8 : 4;
    const long long d = c->channels, all = (long long)c->batch * d * c->states;
    auto area = [&](const char* n, const Rows& rows) { return strided(n, rows, c->batch, c->len, es); };
    const Area outs[] = {area("dx", w[0]), area("ddt", w[1]), area("dz", w[2]), area("dB", w[3]), area("dC", w[4]), packed("dA", dA, d * c->states, as),
                         packed("dD", dD, d, as), packed("ddt_bias", ddt_bias, d, as), packed("dh_in", dh_in, all, as),
                         packed("ws", ws, rp_selective_scan_ws_bytes(c, dtype, 1) / (long long)as, as)};
    const Area ins[] = {area("dy", r.y), area("x", r.x), area("dt", r.dt), area("B", r.B), area("C", r.C), area("z", r.z),
                        packed("A", A, d * c->states, as), packed("D", D, d, as), packed("dt_bias", dt_bias, d, as), packed("dh_out", dh_out, all, as),
                        packed("saved", saved, rp_selective_scan_saved_elems(c, dtype), as), packed("lengths", lengths, c->batch, sizeof(int))};
    if (refuse_buffers(name, outs, ins)) return -1;
    DeviceScope scope;
    if (scope.enter(device_id)) return refuse(name, "no such device");
    const Wanted want = {dx, ddt, dA, dB, dC, dD, ddt_bias, dz, dh_in, accumulate};
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return by_type(dtype, [&](auto t) {
        return by_lanes(c->states, c->channels / c->groups, [&](auto p, auto pads) { return backward_p<decltype(t), decltype(p)::value, decltype(pads)::value>(want, dy, dh_out, o, saved, ws, c, s); });
    });
}

}  // extern "C"
