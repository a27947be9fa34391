// token_attention_general.cuh -- token attention for every type, stride and
// head width: one tile of TL x TL scores at a time in registers, operands in
// shared memory in the accumulator type, products on the FMA pipes.  This is
// the path of fp32 and fp64 tensors (whose products the tensor cores would
// round) and of layouts that a TMA box cannot describe.
//
// A thread (tx, ty) of the 16 x 16 block owns score rows ty + 16 i and
// columns tx + 16 j; tiles are padded by four elements a row, so the 16-byte
// reads of eight neighbouring rows fall in different banks.  Per four
// channels a thread reads 2 MI vectors for 4 MI^2 multiply-adds.
#pragma once

#include <cfloat>

#include "token_attention.h"

namespace nsc {
namespace tok {

constexpr int kGenThreads = 256;

template <typename A> __device__ __forceinline__ A ninf() { return -INFINITY; }
__device__ __forceinline__ float exp2_(float x) { return exp2f(x); }
__device__ __forceinline__ double exp2_(double x) { return exp2(x); }
__device__ __forceinline__ float log2_(float x) { return log2f(x); }
__device__ __forceinline__ double log2_(double x) { return log2(x); }
__device__ __forceinline__ float tanh_(float x) { return tanhf(x); }
__device__ __forceinline__ double tanh_(double x) { return tanh(x); }

template <typename T> __device__ __forceinline__ T store_as(float v) { return from_float<T>(v); }
template <typename T> __device__ __forceinline__ T store_as(double v) { return v; }

template <int DP, int TL>
struct GenTile {
    static constexpr int MI = TL / 16;              // rows (and columns) of a thread
    static constexpr int LD = DP + 4;               // shared row stride
    static constexpr int VEC = DP >= 64 ? 4 : DP / 16;
    static constexpr int NG = DP / (16 * VEC);      // channel groups of a thread
    static constexpr int LP = TL + 4;
};

// Rows [r0, r0 + TL) of one head into shared memory as A; rows outside
// [lo, hi) and channels past D are zero.  Returns whether this thread saw a
// value that is not finite.
template <typename T, typename A, int DP, int TL>
__device__ __forceinline__ bool load_tile(A* dst, const T* src, int64_t row_stride, int r0, int lo,
                                          int hi, int D) {
    using G = GenTile<DP, TL>;
    bool odd = false;
    for (int i = threadIdx.x; i < TL * DP; i += kGenThreads) {
        const int r = i / DP, d = i % DP, row = r0 + r;
        A v = 0;
        if (row >= lo && row < hi && d < D) {
            v = to_acc(src[row * row_stride + d]);
            odd |= !(v - v == A(0));
        }
        dst[r * G::LD + d] = v;
    }
    return odd;
}

// acc[i][j] = sum_d a[ty + 16 i][d] b[tx + 16 j][d]
template <typename A, int DP, int TL>
__device__ __forceinline__ void dot_tile(const A* a, const A* b, int tx, int ty,
                                         A (&acc)[TL / 16][TL / 16]) {
    using G = GenTile<DP, TL>;
#pragma unroll
    for (int i = 0; i < G::MI; ++i)
#pragma unroll
        for (int j = 0; j < G::MI; ++j) acc[i][j] = 0;
#pragma unroll 2
    for (int d = 0; d < DP; d += 4) {
        A x[G::MI][4], y[G::MI][4];
#pragma unroll
        for (int i = 0; i < G::MI; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[i][e] = a[(ty + 16 * i) * G::LD + d + e];
                y[i][e] = b[(tx + 16 * i) * G::LD + d + e];
            }
#pragma unroll
        for (int i = 0; i < G::MI; ++i)
#pragma unroll
            for (int j = 0; j < G::MI; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j] += x[i][e] * y[j][e];
    }
}

// out[i][g][e] += sum_k w[ty + 16 i][k] b[k][channel]; with `strict` a zero
// weight contributes nothing even where b is not finite (a masked value).
template <typename A, int DP, int TL>
__device__ __forceinline__ void mix_tile(const A* w, const A* b, int tx, int ty, bool strict,
                                         A (&out)[TL / 16][GenTile<DP, TL>::NG]
                                                 [GenTile<DP, TL>::VEC]) {
    using G = GenTile<DP, TL>;
    if (strict) {
        for (int k = 0; k < TL; ++k)
#pragma unroll
            for (int i = 0; i < G::MI; ++i) {
                const A x = w[(ty + 16 * i) * G::LP + k];
                if (x == A(0)) continue;
#pragma unroll
                for (int g = 0; g < G::NG; ++g)
#pragma unroll
                    for (int e = 0; e < G::VEC; ++e)
                        out[i][g][e] += x * b[k * G::LD + (g * 16 + tx) * G::VEC + e];
            }
        return;
    }
#pragma unroll 1
    for (int k = 0; k < TL; k += 4) {
        A x[G::MI][4];
#pragma unroll
        for (int i = 0; i < G::MI; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][e] = w[(ty + 16 * i) * G::LP + k + e];
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int g = 0; g < G::NG; ++g) {
                A y[G::VEC];
#pragma unroll
                for (int e = 0; e < G::VEC; ++e)
                    y[e] = b[(k + kk) * G::LD + (g * 16 + tx) * G::VEC + e];
#pragma unroll
                for (int i = 0; i < G::MI; ++i)
#pragma unroll
                    for (int e = 0; e < G::VEC; ++e) out[i][g][e] += x[i][kk] * y[e];
            }
    }
}

// The bias of every clamped distance for head h, and its bucket.
template <typename A>
__device__ __forceinline__ void load_bias(const Params& p, int h, A* bias) {
    for (int i = threadIdx.x; i <= 2 * p.reach; i += kGenThreads)
        bias[i] = bias2_at<A>(p, __ldg(p.lut + i), h);
}
__device__ __forceinline__ int distance_at(const Params& p, int rel) {
    return min(max(rel, -p.reach), p.reach) + p.reach;
}

// Smallest lo and largest hi over the block's rows that see anything.
__device__ __forceinline__ void join_spans(int lo, int hi, int* box, int& first, int& last) {
    if (threadIdx.x == 0) { box[0] = INT_MAX; box[1] = 0; }
    __syncthreads();
    if (hi > lo) {
        atomicMin(box, lo);
        atomicMax(box + 1, hi);
    }
    __syncthreads();
    last = box[1];
    first = last ? box[0] : 0;   // (no row sees anything: 0, 0)
}

template <typename A, int DP, int TL>
size_t gen_smem(int tiles, int weights, int reach_entries) {
    using G = GenTile<DP, TL>;
    return sizeof(A) * (static_cast<size_t>(tiles) * TL * G::LD +
                        static_cast<size_t>(weights) * TL * G::LP + reach_entries);
}

// f<T, A, DP, TL>() for a dtype, a head width and a tile of 64 or 32 (general_tile).
#define NSC_GEN_WIDTHS(F, T, A)                                       \
    (p.D > 128 ? F<T, A, 256, 32>(NSC_GEN_ARGS)                       \
     : tile == 32 ? (p.D <= 32 ? F<T, A, 32, 32>(NSC_GEN_ARGS)        \
                     : p.D <= 64 ? F<T, A, 64, 32>(NSC_GEN_ARGS)      \
                                 : F<T, A, 128, 32>(NSC_GEN_ARGS))    \
     : p.D <= 32 ? F<T, A, 32, 64>(NSC_GEN_ARGS)                      \
     : p.D <= 64 ? F<T, A, 64, 64>(NSC_GEN_ARGS)                      \
                 : F<T, A, 128, 64>(NSC_GEN_ARGS))
#define NSC_GEN_DISPATCH(F)                                           \
    const int tile = general_tile(dtype, p.B, p.Hkv, p.Lq, p.Lk, p.D); \
    switch (dtype) {                                                  \
        case NSC_F16: return NSC_GEN_WIDTHS(F, __half, float);        \
        case NSC_BF16: return NSC_GEN_WIDTHS(F, __nv_bfloat16, float);\
        case NSC_F32: return NSC_GEN_WIDTHS(F, float, float);         \
        default:                                                      \
            return p.D <= 32 ? F<double, double, 32, 32>(NSC_GEN_ARGS)\
                 : p.D <= 64 ? F<double, double, 64, 32>(NSC_GEN_ARGS)\
                             : F<double, double, 128, 32>(NSC_GEN_ARGS);\
    }

}  // namespace tok
}  // namespace nsc
