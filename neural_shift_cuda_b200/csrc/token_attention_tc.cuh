// token_attention_tc.cuh -- what the tensor-core kernels of token attention
// share: tensor maps of (B, L, H, D) operands, the guard against values that
// are not finite, score arithmetic, and bounded waits.
#pragma once

#include <climits>

#include "nsc_tcgen05.cuh"
#include "token_attention.h"

namespace nsc {
namespace tok {

constexpr int kRows = 128;            // rows of a tile: lanes of tensor memory
constexpr int kPanel = kRows * 128;   // bytes of a panel: 128 rows of 64 16-bit elements
constexpr int kBiasPad = 160;         // distances past the reach that a tile's rows meet

struct Bounded {                      // wait accounting of a launch
    unsigned* timeouts;
    int skip;                         // test hook: a copy left unissued
    unsigned budget;
};

// As mbar_wait32_ab, all in line: a call would have to keep to the caller's
// registers, which the warps of a kernel that shares them out do not have alike.
__device__ __forceinline__ bool wait_bounded(uint64_t* bar, uint32_t parity, unsigned* timeouts,
                                             volatile int* abort_flag) {
    const uint32_t a = smem_u32(bar);
    if (mbar_try_wait32(a, parity)) return true;
    const uint32_t budget = static_cast<uint32_t>(abort_flag[1]);
    for (uint32_t i = 0; i < budget; ++i) {
        if (mbar_try_wait_sleep32(a, parity)) return true;
        if (*abort_flag) return false;
    }
    atomicAdd(timeouts, 1u);
    *abort_flag = 1;
    return false;
}

// Coordinates of a (B, L, H, D) tensor map: {D, H, L, B}, boxes of 64 channels of `rows` rows.
bool encode_heads(CUtensorMap* map, const void* base, const int64_t* strides, int B, int L, int H,
                  int D, bool bf16, const char** err, int rows = kRows);

template <typename T, int DP> nsc_status tc_fwd_run(const Params& p, cudaStream_t st);
template <typename T, int DP>
nsc_status tc_bwd_run(const Params& p, const Grads& g, const void* recs, cudaStream_t st);

// A query row as the backward kernels read it: the forward's statistics (m NaN
// where delta is not finite), delta, and the norm of its output gradient.
struct RowRec { float m, ll, delta, norm; };
constexpr int kRecRows = 128;  // rows of a record block, and of one entry of their largest norms

// Every fourth row (from the part-th) of [lo, hi) of n, rows of a whole record block at once.
template <typename One, typename Block>
__device__ __forceinline__ void over_span(int lo, int hi, int n, int part, One one, Block block) {
    const int first = (lo + kRecRows - 1) / kRecRows;
    const int last = hi == n ? (n + kRecRows - 1) / kRecRows : hi / kRecRows;   // (the end's is whole)
    const int a = first < last ? first * kRecRows : hi, b = first < last ? last * kRecRows : hi;
    for (int i = first + part; i < last; i += 4) block(i);
    for (int i = lo + part; i < a; i += 4) one(i);
    for (int i = b + part; i < hi; i += 4) one(i);
}

// A tile: ROWS rows from `row` of head `h`, DP / 64 panels.
template <int DP, int ROWS = kRows>
__device__ __forceinline__ void load_rows(unsigned char* dst, const CUtensorMap* map, uint64_t* bar,
                                          int h, int row, int b) {
#pragma unroll
    for (int c = 0; c < DP / 64; ++c) tma_load_4d(dst + c * ROWS * 128, map, bar, 64 * c, h, row, b);
}

// Bits [lo, hi) of 32, for any lo and hi.
__device__ __forceinline__ uint32_t seen_bits(int lo, int hi) {
    const int l = min(max(lo, 0), 32), h = min(max(hi, 0), 32);
    const uint32_t below_h = h == 32 ? ~0u : (1u << h) - 1, below_l = l == 32 ? ~0u : (1u << l) - 1;
    return below_h & ~below_l;
}

// Sees to it that rows of a landed tile that hold an infinity or NaN do not
// reach products as anything but zero: a weight of zero does not hide them.
// `lanes` threads, thread t has rows t, t + lanes, ...; returns a bit for each of
// its rows (in that order) that held such a value.  x 0 is 0 or NaN, so one
// multiply-add per two values finds them.
template <typename T, int DP, int ROWS = kRows>
__device__ __forceinline__ uint32_t scrub_rows(unsigned char* tile, int t, int lanes) {
    uint32_t bad = 0;
    int bit = 0;
    for (int r = t; r < ROWS; r += lanes, ++bit) {
        using T2 = typename std::conditional<sizeof(T) == 2 && std::is_same<T, __half>::value,
                                             __half2, __nv_bfloat162>::type;
        T2 zero, acc[4];   // (four: one chain would wait out each step)
        reinterpret_cast<uint32_t&>(zero) = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = zero;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            const uint4* row = reinterpret_cast<const uint4*>(tile + c * ROWS * 128 + r * 128);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint4 v = row[(i + r) & 7];
                acc[0] = __hfma2(reinterpret_cast<const T2&>(v.x), zero, acc[0]);
                acc[1] = __hfma2(reinterpret_cast<const T2&>(v.y), zero, acc[1]);
                acc[2] = __hfma2(reinterpret_cast<const T2&>(v.z), zero, acc[2]);
                acc[3] = __hfma2(reinterpret_cast<const T2&>(v.w), zero, acc[3]);
            }
        }
        uint32_t w = 0;   // zeros (of either sign), or NaN
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= reinterpret_cast<const uint32_t&>(acc[i]);
        if ((w & 0x7FFF7FFFu) == 0) continue;
        bad |= 1u << bit;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            uint4* row = reinterpret_cast<uint4*>(tile + c * ROWS * 128 + r * 128);
#pragma unroll
            for (int i = 0; i < 8; ++i) row[i] = make_uint4(0, 0, 0, 0);
        }
    }
    return bad;
}
// Fills row r of a tile with NaN.
template <int DP, int ROWS = kRows>
__device__ __forceinline__ void poison_row(unsigned char* tile, int r) {
#pragma unroll
    for (int c = 0; c < DP / 64; ++c) {
        uint4* row = reinterpret_cast<uint4*>(tile + c * ROWS * 128 + r * 128);
#pragma unroll
        for (int i = 0; i < 8; ++i) row[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
    }
}
__device__ __forceinline__ void fence_async_shared() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// The cap, f tanh(y1 s) of 32 products s, in place.  Up to |y| = 1, tanh y is an odd
// polynomial y P(y^2), P of least maximum error of y P(y^2) against tanh y by
// exchange: 2.4e-7 with six terms (fp16), 2.8e-6 with five (bf16: at a cap of 50,
// 1.4e-4 of a softmax weight that is rounded to 4e-3).  Under caps in the thousands, of
// which scores are a small part, that is 4.2e-5 of each score (its slope at zero is short by
// it): lse is off by as much of itself, weights by as much of a difference of two scores.
// Up to |y| = 0.45, where most scores of a layer lie, two terms less do as well (9e-8 and
// 2.7e-6; 32 heads of 128, 4096 causal tokens 192 -> 179 us in short runs, 205 -> 193 under
// sustained load).  It runs on the FMA pipe, beside the exponentials, in pairs, with y1 and
// f in the coefficients; the hardware's tanh would be one more exponential's time, with 5e-4 of
// error.  A warp with a larger |y| in the chunk takes tanh |y| = 1 - 2 / (1 + e^(2|y|)).
template <typename T> struct Cap {
    static constexpr int N = std::is_same<T, __half>::value ? 6 : 5;
    float c[N], near[N - 2], y1, f, unit;   // |s| = unit at |y| = 1
    __device__ __forceinline__ Cap(float y1_, float f_) : y1(y1_), f(f_) {
        constexpr float k6[6] = {0.9999968539f, -0.3332400381f, 0.1325352535f,
                                 -0.05097286522f, 0.01611418278f, -0.002839466166f};
        constexpr float k5[6] = {0.9999684695f, -0.3326582321f, 0.1292206686f,
                                 -0.04329986371f, 0.008365886550f, 0.f};
        constexpr float k4[4] = {0.9999989514f, -0.3332630012f, 0.1320517446f, -0.045149514f};
        constexpr float k3[4] = {0.9999585229f, -0.3316544208f, 0.1160969438f, 0.f};
        float y = y1 * f;
#pragma unroll
        for (int i = 0; i < N; ++i, y *= y1 * y1) {
            c[i] = (N == 6 ? k6[i] : k5[i]) * y;
            if (i < N - 2) near[i] = (N == 6 ? k4[i % 4] : k3[i % 4]) * y;
        }
        unit = y1 != 0.f ? 1.f / fabsf(y1) : INFINITY;
    }
    template <int M> static __device__ __forceinline__ void odd(float2* s, const float (&k)[M]) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 u = __fmul2_rn(s[i], s[i]);
            float2 p = make_float2(k[M - 1], k[M - 1]);
#pragma unroll
            for (int j = M - 2; j >= 0; --j) p = __ffma2_rn(p, u, make_float2(k[j], k[j]));
            s[i] = __fmul2_rn(s[i], p);
        }
    }
    __device__ __forceinline__ void operator()(float2* s) const {
        float top[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i)
            top[i & 3] = fmaxf(top[i & 3], fmaxf(fabsf(s[i].x), fabsf(s[i].y)));
        top[0] = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        if (!__any_sync(0xffffffffu, top[0] > 0.45f * unit)) {
            odd<N - 2>(s, near);
            return;
        }
        if (!__any_sync(0xffffffffu, top[0] > unit)) {
            odd<N>(s, c);
            return;
        }
        float* v = reinterpret_cast<float*>(s);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const float y = v[i] * y1;
            const float e = tc::ex2(fabsf(y) * static_cast<float>(2 * kLog2e));
            v[i] = copysignf(f - __fdividef(2.f * f, 1.f + e), y);
        }
    }
};

// Bias of head h by clamped distance, with kBiasPad more of the end values at
// each end: E[distance + reach + kBiasPad].
__device__ __forceinline__ void load_padded_bias(const Params& p, int h, float* E, int t, int n) {
    for (int i = t; i <= 2 * p.reach + 2 * kBiasPad; i += n) {
        const int d = min(max(i - kBiasPad, 0), 2 * p.reach);
        E[i] = bias2_at<float>(p, __ldg(p.lut + d), h);
    }
}

// The products of two tiles, issued by one lane of a converged warp.  scores_mma:
// [128 x N] = A B^T over the channels, A of 128 rows and B of N, both K-major; `steps` of
// 16 channels.  mix_mma: [128 x channels] += W B with the weights W (128 x 16 K) in tensor
// memory, RUN k-steps side by side and GAP columns from one such run to the next, and the
// 16 K rows of B, in panels of `panel` bytes, as the reduced dimension.
template <int DP, int N = kRows>
__device__ __forceinline__ void scores_mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                           int steps) {
    const uint32_t x = tc::operand(a, 16), y = tc::operand(b, 16);
#pragma unroll
    for (int c = 0; c < DP / 16; ++c)
        if (c < steps)
            tc::mma_ss(d, x + (((c >> 2) * kPanel + (c & 3) * 32) >> 4),
                       y + (((c >> 2) * N * 128 + (c & 3) * 32) >> 4), idesc, c > 0);
}
template <int K, int RUN, int GAP>
__device__ __forceinline__ void mix_mma(uint32_t d, uint32_t w, uint32_t b, uint32_t panel,
                                        uint32_t idesc, bool add) {
    const uint32_t y = tc::operand(b, panel);
#pragma unroll
    for (int k = 0; k < K; ++k)
        tc::mma_ts(d, w + k / RUN * GAP + k % RUN * 8, y + ((k * 2048) >> 4), idesc, add || k > 0);
}

}  // namespace tok
}  // namespace nsc
