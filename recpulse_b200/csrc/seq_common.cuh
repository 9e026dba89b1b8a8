/* Shared by the operators along a sequence (causal_conv.cu, selective_scan.cu, block_norm.cu): element types and
 * their accumulators, vectors of channels, device selection. */
#ifndef RPB_SEQ_COMMON_CUH
#define RPB_SEQ_COMMON_CUH

#include <cstdio>
#include <cstring>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "rpb_common.h"

extern "C" void rpb_count_launches(int n);      /* gemm_dispatch.cu */

namespace rpb_seq {

#define SEQ_CUDA(call)                                                                          \
    do {                                                                                        \
        cudaError_t e_ = (call);                                                                \
        if (e_ != cudaSuccess) {                                                                \
            fprintf(stderr, "recpulse_b200: %s failed: %s\n", #call, cudaGetErrorString(e_));   \
            return -1;                                                                          \
        }                                                                                       \
    } while (0)

/* Sums, states and statistics are held in float, in double for float64. */
template <typename T> struct AccOf { typedef float type; };
template <> struct AccOf<double> { typedef double type; };

template <typename T> __device__ __forceinline__ typename AccOf<T>::type up(T v) { return (typename AccOf<T>::type)v; }
template <> __device__ __forceinline__ float up<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float up<__half>(__half v) { return __half2float(v); }
template <typename T, typename A> __device__ __forceinline__ T down(A v) { return (T)v; }
template <> __device__ __forceinline__ __nv_bfloat16 down<__nv_bfloat16, float>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half down<__half, float>(float v) { return __float2half_rn(v); }

/* V consecutive channels of one row, as they lie in memory. */
template <typename T, int V> struct alignas((sizeof(T) * V) < 16 ? sizeof(T) * V : 16) Pack {
    T v[V];
};

template <typename T, int V> __device__ __forceinline__ Pack<T, V> zero_pack() {
    Pack<T, V> p;
#pragma unroll
    for (int i = 0; i < V; ++i) p.v[i] = down<T>(typename AccOf<T>::type(0));
    return p;
}

/* V sums rounded to the stored type, two at a time where the type is half as wide */
template <typename T, int V, typename A> __device__ __forceinline__ Pack<T, V> narrow(const A (&v)[V]) {
    Pack<T, V> p;
#pragma unroll
    for (int i = 0; i < V; ++i) p.v[i] = down<T>(v[i]);
    return p;
}
template <int V> __device__ __forceinline__ Pack<__nv_bfloat16, V> narrow_pairs(const float (&v)[V], __nv_bfloat16) {
    Pack<__nv_bfloat16, V> p;
#pragma unroll
    for (int i = 0; i < V; i += 2) *reinterpret_cast<__nv_bfloat162*>(&p.v[i]) = __floats2bfloat162_rn(v[i], v[i + 1]);
    return p;
}
template <int V> __device__ __forceinline__ Pack<__half, V> narrow_pairs(const float (&v)[V], __half) {
    Pack<__half, V> p;
#pragma unroll
    for (int i = 0; i < V; i += 2) *reinterpret_cast<__half2*>(&p.v[i]) = __floats2half2_rn(v[i], v[i + 1]);
    return p;
}
template <typename T, int V, typename A> __device__ __forceinline__ Pack<T, V> store_form(const A (&v)[V]) {
    if constexpr (sizeof(T) == 2 && V % 2 == 0) return narrow_pairs<V>(v, T());
    else return narrow<T, V>(v);
}

/* Reads `valid` (<= V, may be <= 0) channels at p, zeros behind them; `vec`: p is aligned for the whole pack. */
template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_pack(const T* p, int valid, bool vec) {
    if (vec && valid >= V) return *reinterpret_cast<const Pack<T, V>*>(p);
    Pack<T, V> r = zero_pack<T, V>();
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < valid) r.v[i] = p[i];
    return r;
}
template <typename T, int V> __device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& r, int valid, bool vec) {
    if (vec && valid >= V) { *reinterpret_cast<Pack<T, V>*>(p) = r; return; }
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < valid) p[i] = r.v[i];
}

__device__ __forceinline__ float ex2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
/* two floats in one 64-bit register pair: one instruction for two multiplications or multiply-adds */
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

/* exp(v) through the hardware's base-2 exponential, results below the normal range as 0: within (2 + |v|) steps */
__device__ __forceinline__ float exp_of(float v) { return ex2_fast(v * 1.44269504088896341f); }
__device__ __forceinline__ float reciprocal(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

/* 1 / (1 + exp(-v)); the reciprocal of +inf is 0, so both ends are exact */
__device__ __forceinline__ float logistic(float v) { return reciprocal(1.0f + exp_of(-v)); }
__device__ __forceinline__ double logistic(double v) { return 1.0 / (1.0 + exp(-v)); }

/* log(1 + exp(v)) = max(v, 0) + log(1 + e) with e = exp(-|v|) in (0, 1]; log(1 + e) / e as a polynomial of degree 9
 * (Chebyshev interpolation on [0, 1]), within 2.2 half-steps of float32 for the e that it is given: a third of log1pf's instructions,
 * and no cancellation for small e.  e carries exp_of's error, which for v far below 0, where the result is e, is the result's: within
 * (2 + |v|) steps more */
__device__ __forceinline__ float softplus_of(float v) {
    const float e = exp_of(-fabsf(v));
    float p = -0.0031760570127516985f;
    p = fmaf(p, e, 0.019542528316378593f);
    p = fmaf(p, e, -0.05637361481785774f);
    p = fmaf(p, e, 0.10543623566627502f);
    p = fmaf(p, e, -0.1526966691017151f);
    p = fmaf(p, e, 0.1966327428817749f);
    p = fmaf(p, e, -0.24951615929603577f);
    p = fmaf(p, e, 0.33329710364341736f);
    p = fmaf(p, e, -0.49999892711639404f);
    p = fmaf(p, e, 1.0f);
    return fmaf(p, e, fmaxf(v, 0.0f));
}
__device__ __forceinline__ double softplus_of(double v) { return fmax(v, 0.0) + log1p(exp(-fabs(v))); }

/* softplus of V values: in float two at a time */
template <int V> __device__ __forceinline__ void softplus_all(double (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = softplus_of(v[i]);
}
template <int V> __device__ __forceinline__ void softplus_all(float (&v)[V]) {
    if (V % 2) v[V - 1] = softplus_of(v[V - 1]);
#pragma unroll
    for (int i = 0; i < V / 2 * 2; i += 2) {
        const f32x2 e = pack2(exp_of(-fabsf(v[i])), exp_of(-fabsf(v[i + 1])));
        const float c[9] = {0.019542528316378593f, -0.05637361481785774f, 0.10543623566627502f, -0.1526966691017151f, 0.1966327428817749f,
                            -0.24951615929603577f, 0.33329710364341736f, -0.49999892711639404f, 1.0f};
        f32x2 p = pack2(-0.0031760570127516985f, -0.0031760570127516985f);
#pragma unroll
        for (int k = 0; k < 9; ++k) p = fma2(p, e, pack2(c[k], c[k]));
        unpack2(fma2(p, e, pack2(fmaxf(v[i], 0.0f), fmaxf(v[i + 1], 0.0f))), v[i], v[i + 1]);
    }
}

/* Asynchronous copies into shared memory: the first `size` of BYTES bytes (nothing is read for 0), zeros for the rest. */
template <int BYTES> __device__ __forceinline__ void async_copy_part(void* to, const void* from, int size) {
    const unsigned dst = (unsigned)__cvta_generic_to_shared(to);
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(from), "r"(size) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(from), "n"(BYTES), "r"(size) : "memory");
}
template <int BYTES> __device__ __forceinline__ void async_copy(void* to, const void* from, bool on) { async_copy_part<BYTES>(to, from, on ? BYTES : 0); }
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }


/* Runs a call on the tensors' device and gives the caller's current device back. */
struct DeviceScope {
    int prev = -1; bool moved = false;
    int enter(int device) {
        if (cudaGetDevice(&prev) != cudaSuccess) return -1;
        if (prev != device) { if (cudaSetDevice(device) != cudaSuccess) return -1; moved = true; }
        return 0;
    }
    ~DeviceScope() { if (moved) cudaSetDevice(prev); }
};

/* Lets a kernel use `bytes` of dynamic shared memory on the current device; the driver is asked once per kernel and device. */
template <typename K> int allow_shared(K kernel, size_t bytes, int device, unsigned char (&done)[64]) {
    if (bytes <= 40 * 1024 || (device < 64 && done[device])) return 0;
    SEQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024));
    if (device < 64) done[device] = 1;
    return 0;
}

inline int refuse(const char* what, const char* why) {
    fprintf(stderr, "recpulse_b200: %s: %s\n", what, why);
    return -1;
}

/* A strided [batch, len, channels] operand with unit channel stride, for the host's checks. */
struct Rows { const void* p; long long batch, row, channels; };

/* Strides of such an operand that is READ: rows of at least `channels` elements; a batch stride of 0 (one sequence for
 * all) is allowed.  Strides that no index uses (one row, one sequence) may be anything. */
inline bool readable(const Rows& r, int batch, int len) {
    return (len == 1 || r.row >= r.channels) && (batch == 1 || r.batch >= 0);
}
/* ... and of one that is WRITTEN: no two elements at one address, sequences one after the other or row by row in turn. */
inline bool writable(const Rows& r, int batch, int len) {
    if (len > 1 && r.row < r.channels) return false;
    if (batch == 1) return true;
    if (len == 1) return r.batch >= r.channels;
    return r.batch >= (len - 1) * r.row + r.channels || (r.batch >= r.channels && r.row >= (batch - 1) * r.batch + r.channels);
}
/* Whether packs of `bytes` bytes can be moved at every row of the operand. */
inline bool aligned_rows(const Rows& r, int batch, int len, size_t es, size_t bytes) {
    const long long size = (long long)es, step = (long long)bytes;
    return (reinterpret_cast<uintptr_t>(r.p) % bytes) == 0 && (batch == 1 || r.batch * size % step == 0) && (len == 1 || r.row * size % step == 0);
}

/* What a call reads or writes, for the host's checks of overlaps: a strided operand, or a packed one as a single row. */
struct Area {
    const char* name;
    Rows r;
    int batch, len;
    long long size;             /* bytes per element */
    const void* in_place;       /* an operand that this output may be, or NULL */
};
inline Area strided(const char* name, const Rows& r, int batch, int len, size_t size) { return {name, r, batch, len, (long long)size, nullptr}; }
inline Area packed(const char* name, const void* p, long long elems, size_t size, const void* in_place = nullptr) {
    return {name, {elems > 0 ? p : nullptr, 0, 0, elems}, 1, 1, (long long)size, in_place};
}

/* Whether two of them share a byte.  Column blocks of one buffer (the halves of a projection's output) do not; where that cannot
 * be seen from the strides, operands whose extents meet count as sharing. */
inline bool overlaps(const Area& a, const Area& b) {
    if (!a.r.p || !b.r.p) return false;
    const char *a0 = reinterpret_cast<const char*>(a.r.p), *b0 = reinterpret_cast<const char*>(b.r.p);
    const char* a1 = a0 + ((a.batch - 1) * a.r.batch + (a.len - 1) * a.r.row + a.r.channels) * a.size;
    const char* b1 = b0 + ((b.batch - 1) * b.r.batch + (b.len - 1) * b.r.row + b.r.channels) * b.size;
    if (a1 <= b0 || b1 <= a0) return false;
    const bool a_single = a.batch == 1 && a.len == 1, b_single = b.batch == 1 && b.len == 1;
    if (a_single && b_single) return true;
    if (a_single) return overlaps(b, a);
    const long long unit = a.len > 1 ? a.r.row : a.r.batch;     /* every row of a (of both, if b has several) begins a multiple of it from its base */
    if (unit <= 0 || (a.batch > 1 && a.r.batch % unit != 0)) return true;
    if (!b_single && (a.size != b.size || (a.len > 1 && a.r.row != b.r.row) || (a.batch > 1 && b.r.batch % unit != 0))) return true;
    const long long apart = (b0 - a0) % (unit * a.size);
    const long long shift = apart < 0 ? apart + unit * a.size : apart;
    return !(shift >= a.r.channels * a.size && shift + b.r.channels * b.size <= unit * a.size);
}

/* Whether the elements lie on boundaries of their size: the GPU faults on others. */
inline bool on_boundaries(const Area& a) { return reinterpret_cast<uintptr_t>(a.r.p) % (uintptr_t)a.size == 0; }

/* Refuses buffers off their elements' boundaries, and outputs that share memory with what the call reads or with one another. */
template <int N, int M> int refuse_buffers(const char* what, const Area (&outs)[N], const Area (&ins)[M]) {
    for (int i = 0; i < N + M; ++i) {
        const Area& a = i < N ? outs[i] : ins[i - N];
        if (on_boundaries(a)) continue;
        fprintf(stderr, "recpulse_b200: %s: %s is not aligned to its elements\n", what, a.name);
        return -1;
    }
    for (int i = 0; i < N; ++i) {
        for (int k = 0; k < M; ++k)
            if (!(outs[i].in_place && outs[i].r.p == outs[i].in_place && ins[k].r.p == outs[i].in_place) && overlaps(outs[i], ins[k])) {
                fprintf(stderr, "recpulse_b200: %s: %s overlaps %s\n", what, outs[i].name, ins[k].name);
                return -1;
            }
        for (int k = 0; k < i; ++k)
            if (overlaps(outs[i], outs[k])) {
                fprintf(stderr, "recpulse_b200: %s: %s overlaps %s\n", what, outs[i].name, outs[k].name);
                return -1;
            }
    }
    return 0;
}

constexpr int SM_COUNT = 148;       /* of the one chip this library is written for; sizes of splits follow it */

/* Sums of partial results, parts x columns, into up to three outputs: out[c] (+)= sum over parts, in a fixed order
 * (each of 8 threads every eighth part, then the eight sums in turn), so equal inputs give equal bits. */
struct PartSums {
    void* out[3];                   /* NULL: not wanted */
    long long first[3], cols[3];    /* the output's columns within a part */
    int accumulate[3];
    int blocks[3];
};

template <typename T>
__global__ void __launch_bounds__(256) sum_parts_kernel(PartSums d, const typename AccOf<T>::type* __restrict__ parts, int n_parts,
                                                        long long part_stride) {
    typedef typename AccOf<T>::type A;
    __shared__ A sums[8][33];
    rpb_pdl_trigger();
    rpb_pdl_wait();
    int k = 0;
    long long block = blockIdx.x;
    while (k < 2 && block >= d.blocks[k]) block -= d.blocks[k++];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const long long col = block * 32 + tx;
    A s = 0;
    if (col < d.cols[k]) {
        const A* p = parts + d.first[k] + col;
#pragma unroll 8
        for (int i = ty; i < n_parts; i += 8) s += p[i * part_stride];
    }
    sums[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && col < d.cols[k]) {
#pragma unroll
        for (int i = 1; i < 8; ++i) s += sums[i][tx];
        T* o = reinterpret_cast<T*>(d.out[k]) + col;
        if (d.accumulate[k]) s += up(*o);
        *o = down<T>(s);
    }
}

template <typename T>
int sum_parts(PartSums d, const void* parts, int n_parts, long long part_stride, cudaStream_t s) {
    typedef typename AccOf<T>::type A;
    long long blocks = 0;
    for (int k = 0; k < 3; ++k) {
        d.blocks[k] = d.out[k] ? (int)((d.cols[k] + 31) / 32) : 0;
        blocks += d.blocks[k];
    }
    if (blocks == 0) return 0;
    SEQ_CUDA(rpb_launch(sum_parts_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, 1, d, reinterpret_cast<const A*>(parts), n_parts,
                        part_stride));
    rpb_count_launches(1);
    return 0;
}

}  // namespace rpb_seq

#endif
