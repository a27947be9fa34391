// token_attention_tc_bwd.cuh -- backward of token attention on the tensor
// cores, fp16 / bf16, head widths up to 128.  The formulas are those of
// token_attention_general_bwd.cu; two kernels, no atomics.
//
// tc_dkv_kernel keeps 128 keys in place and passes the query tiles of every head
// that shares the key head.  It works transposed (S^T = K Q^T, dP^T = V dO^T: a
// thread's lane is a key), so that P^T and dS^T are left in tensor memory as the
// A operands of dV = P^T dO and dK = dS^T Q, and Q and dO serve each as both
// kinds of operand from one landed tile.  512 threads take a quarter of a row
// each, in two phases: P from S, then dS from dP.  The products of one phase run beside
// the other: dV(i), S(i+1) beside phase two of i, dK(i), dP(i+1) beside phase one of
// i+1; one warp issues S and dP, another dV and dK (one warp for all was late for both:
// 5 % of the time with heads of 64).  Tensor memory is full at D = 128 (S, dP, dK, dV);
// with heads of 64 there are two S, so that S(i+1) need not wait for dV(i).
//
// tc_dq_kernel keeps 128 queries in place: S, dP, then dQ += dS K with dS in the
// place of its S.  S has two buffers and dP is free once it is in registers, so
// S(j+1) and dP(j+1) run beside the arithmetic of block j.  Recomputing the
// scores here costs two of seven products and buys sums in one order without
// an fp32 gradient in memory.
//
// dS is a product's operand of 16 bits twice: rounded, and what that rounding dropped
// (grad_q and grad_k 2.7e-3 -> 1.7e-3 off in bf16, which is their own rounding, for a
// tenth of the time).  P is rounded once, as in the forward.
//
// Bounded by the arithmetic between the products: 16384 scores a tile on 128 lanes, some
// 20 instructions each (30 with a cap), against 20 D clocks (dkv) and 16 D (dq) of the
// tensor pipe, of which only part runs beside it; a block's set-up and end are some 6 us
// of 35.  4 x 2048 tokens, 16 heads of 64, bias table, bf16: dkv 246 us, dq 252 us (4 and 3
// products of 34 GF: 559 and 409 TF/s).  8192 tokens in 4 documents, causal, capped,
// 16 / 4 heads of 128: dkv 381 us, dq 268 us.
//
// fp16: weights and score gradients of long rows lie below its normal range, and those of
// large values or large gradients of lse above it.  P is held times 2^6, and P (dP - delta)
// over a power of two g that bounds it: |dP - delta| <= |dO| |v| + |delta|, with the largest
// norm of the values that the query sees (dq), or the largest |dO| and |delta| of the
// queries that see the key (dkv).  Each lane, a query or a key, has a g of its own from
// what it sees alone; products are then below 2^14.  Both factors are undone in fp32 at the end.
#pragma once

#include "token_attention_tc.cuh"

namespace nsc {
namespace tok {
namespace {

constexpr int kBwdMath = 512;      // 16 warps of arithmetic, a quarter of a row a thread
constexpr int kBwdThreads = kBwdMath + 128;
constexpr int kMathRegs = 104, kOtherRegs = 64;
constexpr float kPShift = 6.f;   // fp16: log2 of the factor of P

template <int DP> struct BwdShape {
    static constexpr int tile = DP / 64 * kPanel;
    static constexpr int stages = DP == 64 ? 4 : 2;
    static constexpr int smem = 2 * tile + stages * 2 * tile;
};

struct BwdBars {
    uint64_t fixed, x_full[4], y_full[4], empty[4], ok[4];
    // (two each where a warp, or the products, may be a step ahead of a slower warp,
    // whose wait or arrival would else be taken for that of the other step)
    uint64_t s_full[2], p_ready[2], ds_ready[2], used_p[2], used_ds[2], dp_full, dp_free, done;
    uint64_t drain[2];
};

// The g of score gradients whose factor beside P is at most v: a power of two above v, over 2^8.
__device__ __forceinline__ float gradient_scale(float v) {
    if (!(v > 0.f) || !(v < INFINITY)) return 1.f;
    const int e = static_cast<int>((__float_as_uint(v) >> 23) & 0xFF) + 1 - 8;
    return __uint_as_float(static_cast<uint32_t>(min(max(e, 20), 246)) << 23);
}
template <typename T, int DP, bool CAP, bool BIAS>
__global__ __launch_bounds__(kBwdThreads, 1) void tc_dkv_kernel(
    const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mo,
    const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const Params p,
    const Grads gr, const RowRec* __restrict__ recs, const int split, const Bounded bnd) {
    using S = BwdShape<DP>;
    constexpr int NS = S::stages;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ unsigned char smem_raw[];
    __shared__ BwdBars bars;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag[2];
    __shared__ int span[4];
    __shared__ float2 tops[kBf16 ? 1 : 4][kRows];   // largest |dO| and |delta| of a quarter of the queries
    // per stage: -m (or -(m + ll) without bias), -ll, -delta
    __shared__ __align__(16) float rows[NS][3][kRows];
    unsigned char* smem = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    unsigned char* Ks = smem;
    unsigned char* Vs = smem + S::tile;
    unsigned char* ring = smem + 2 * S::tile;   // stages of Q, dO
    float* E = reinterpret_cast<float*>(smem + S::smem);

    const int warp = tc::uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    // a cluster of `split` blocks shares the query heads of a key head
    const int64_t BH = static_cast<int64_t>(p.B) * p.Hkv;
    const int64_t unit_id = blockIdx.x / split;
    const int t = static_cast<int>(unit_id / BH), rank = static_cast<int>(blockIdx.x % split);
    const int bh = static_cast<int>(unit_id % BH), b = bh / p.Hkv, hk = bh % p.Hkv;
    const int heads = p.G / split, head0 = hk * p.G + rank * heads;
    const int k0 = t * kRows, off = p.Lk - p.Lq;

    if (threadIdx.x < 4) span[threadIdx.x] = threadIdx.x == 0 || threadIdx.x == 3 ? INT_MAX : 0;
    if (threadIdx.x == 0) {
        mbar_init(&bars.fixed, 1);
        for (int i = 0; i < NS; ++i) {
            mbar_init(&bars.x_full[i], 1);
            mbar_init(&bars.y_full[i], 1);
            mbar_init(&bars.empty[i], 1);
            mbar_init(&bars.ok[i], 32);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.s_full[i], 1);
            mbar_init(&bars.p_ready[i], kBwdMath);
            mbar_init(&bars.ds_ready[i], kBwdMath);
        }
        mbar_init(&bars.dp_full, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.used_p[i], 1);
            mbar_init(&bars.used_ds[i], 1);
        }
        mbar_init(&bars.done, 1);
        mbar_init(&bars.drain[0], 1);
        mbar_init(&bars.drain[1], 1);
        fence_mbar_init();
        abort_flag[0] = 0;
        abort_flag[1] = static_cast<int>(bnd.budget);
    }
    if (warp == 17) tc::tmem_alloc(&tmem_slot, 512);
    __syncthreads();
    const int key = k0 + static_cast<int>(threadIdx.x & 127);
    int lo = 0, hi = 0;
    if (warp < 16) {
        query_span(p, b, key, lo, hi);
        const int v0 = __reduce_min_sync(0xffffffffu, hi > lo ? lo : INT_MAX);
        const int v1 = __reduce_max_sync(0xffffffffu, hi > lo ? hi : 0);
        const int v2 = __reduce_max_sync(0xffffffffu, hi > lo ? lo : 0);
        const int v3 = __reduce_min_sync(0xffffffffu, hi > lo ? hi : INT_MAX);
        if (lane == 0 && warp < 4) {
            atomicMin(&span[0], v0);
            atomicMax(&span[1], v1);
            atomicMax(&span[2], v2);
            atomicMin(&span[3], v3);
        }
    }
    __syncthreads();
    const uint32_t tmem = tc::uniform(tmem_slot);
    const int s_lo = tc::uniform(span[0]), s_hi = tc::uniform(span[1]);
    const int all_lo = tc::uniform(span[2]), all_hi = tc::uniform(span[3]);
    const int fb = s_hi > s_lo ? s_lo / kRows : 0;
    const int lb = s_hi > s_lo ? (s_hi + kRows - 1) / kRows : 0;
    const int nq = lb - fb, total = nq * heads;
    // a key tail past Lk has zero rows of K and V, and sees nothing
    auto guarded = [&](int j) {
        return !(j * kRows >= all_lo && min((j + 1) * kRows, p.Lq) <= all_hi);
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        return wait_bounded(bar, parity, bnd.timeouts, abort_flag);
    };
    auto Q_at = [&](int s) { return ring + s * 2 * S::tile; };
    auto O_at = [&](int s) { return ring + s * 2 * S::tile + S::tile; };
    const int steps = (p.D + 15) / 16, cols = steps * 16;
    // at D <= 64 there is room for two S: S(i+1) need not wait for dV(i) to read P(i)
    constexpr bool kTwoS = DP == 64;
    const uint32_t t_s = tmem, t_dp = tmem + (kTwoS ? 256 : 128);
    const uint32_t t_dv = t_dp + 128, t_dk = t_dv + DP;

    if (warp < 16) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMathRegs));
        const int part = warp >> 2;   // columns 32 part and on
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t at_s0 = t_s + lane_base + 32 * part, at_dp = t_dp + lane_base + 32 * part;
        const float unit = static_cast<float>((p.cap > 0 ? p.cap : p.scale) * kLog2e);
        const float y1 = p.cap > 0 ? static_cast<float>(p.scale / p.cap) : 0.f;
        const Cap<T> cap(y1, unit);
        const float2 u2 = CAP ? make_float2(1.f, 1.f) : make_float2(unit, unit);
        const float2 slope2 = make_float2(-1.f / (unit * unit), -1.f / (unit * unit));   // 1 - tanh^2 = 1 + s^2 slope
        float g = 1.f;
        if (!kBf16) {
            float2 top = make_float2(0.f, 0.f);
            const int n = (p.Lq + kRecRows - 1) / kRecRows;
            for (int u = 0; u < heads && hi > lo; ++u) {
                const int64_t bq = static_cast<int64_t>(b) * p.Hq + head0 + u;
                over_span(lo, hi, p.Lq, part,
                          [&](int i) {
                              const float4 r = __ldg(reinterpret_cast<const float4*>(recs + bq * p.Lq + i));
                              top.x = fmaxf(top.x, r.w);
                              if (fabsf(r.z) < INFINITY) top.y = fmaxf(top.y, fabsf(r.z));
                          },
                          [&](int i) {
                              top.x = fmaxf(top.x, __ldg(gr.row_norms + bq * n + i));
                              top.y = fmaxf(top.y, __ldg(gr.row_deltas + bq * n + i));
                          });
            }
            const int at = threadIdx.x & 127;
            tops[part][at] = top;
            named_sync(1, kBwdMath);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                top = make_float2(fmaxf(top.x, tops[i][at].x), fmaxf(top.y, tops[i][at].y));
            if (hi > lo)
                g = gradient_scale(top.x * __ldg(gr.value_norms + bh * static_cast<int64_t>(p.Lk) + key) +
                                   top.y);
        }
        const float2 g2 = make_float2(1.f / g, 1.f / g);
        bool alive = true;
        int it = 0;
        for (int u = 0; u < heads && nq > 0; ++u) {
            if (BIAS) {   // E of this head, once all are done with the last (a warp
                          // that gave up comes here too)
                named_sync(1, kBwdMath);
                load_padded_bias(p, head0 + u, E, threadIdx.x, kBwdMath);
                named_sync(1, kBwdMath);
            }
            for (int j = fb; alive && j < lb; ++j, ++it) {
                const int st = it % NS;
                const uint32_t at_s = at_s0 + (kTwoS ? 128 * (it & 1) : 0);
                alive = __all_sync(0xffffffffu, wait(&bars.ok[st], (it / NS) & 1) &&
                                                    wait(&bars.s_full[it & 1], (it >> 1) & 1));
                if (!alive) break;
                tc::fence_after();
                float2 s[16];
                tc::load32(at_s, reinterpret_cast<float*>(s));
                tc::wait_ld();
                if (CAP) cap(s);
                const int q0 = j * kRows + 32 * part;
                const float4* m4 = reinterpret_cast<const float4*>(rows[st][0] + 32 * part);
                const float4* l4 = reinterpret_cast<const float4*>(rows[st][1] + 32 * part);
                const bool whole = __all_sync(0xffffffffu, lo <= q0 && hi >= q0 + 32);
                const uint32_t seen = whole ? 0 : seen_bits(lo - q0, hi - q0);
                const int rel0 = key - (q0 + off);   // distance at column 0, one less a column
                const int w0 = __shfl_sync(0xffffffffu, rel0, 0);
                bool far = false;
                float e_far = 0.f;
                if (BIAS) {
                    far = w0 + 31 <= -p.reach || w0 - 31 >= p.reach;
                    if (far) e_far = E[w0 > 0 ? 2 * p.reach + kBiasPad : kBiasPad];
                }
                const float* er = E + rel0 + p.reach + kBiasPad;
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float4 m = m4[i];
                    float2 x0, x1;
                    if (BIAS) {
                        const float4 l = l4[i];
                        float2 b0 = make_float2(e_far, e_far), b1 = b0;
                        if (!far) {
                            b0 = make_float2(er[-4 * i], er[-4 * i - 1]);
                            b1 = make_float2(er[-4 * i - 2], er[-4 * i - 3]);
                        }
                        x0 = __fadd2_rn(__fadd2_rn(__ffma2_rn(s[2 * i], u2, b0), make_float2(m.x, m.y)),
                                        make_float2(l.x, l.y));
                        x1 = __fadd2_rn(__fadd2_rn(__ffma2_rn(s[2 * i + 1], u2, b1), make_float2(m.z, m.w)),
                                        make_float2(l.z, l.w));
                    } else {
                        x0 = __ffma2_rn(s[2 * i], u2, make_float2(m.x, m.y));
                        x1 = __ffma2_rn(s[2 * i + 1], u2, make_float2(m.z, m.w));
                    }
                    float2 p0 = make_float2(tc::ex2(x0.x), tc::ex2(x0.y));
                    float2 p1 = make_float2(tc::ex2(x1.x), tc::ex2(x1.y));
                    if (!whole) {
                        if (!(seen >> (4 * i) & 1)) p0.x = 0.f;
                        if (!(seen >> (4 * i + 1) & 1)) p0.y = 0.f;
                        if (!(seen >> (4 * i + 2) & 1)) p1.x = 0.f;
                        if (!(seen >> (4 * i + 3) & 1)) p1.y = 0.f;
                    }
                    w[2 * i] = tc::pack2<T>(p0.x, p0.y);
                    w[2 * i + 1] = tc::pack2<T>(p1.x, p1.y);
                    if (!kBf16) {   // over g from here on
                        p0 = __fmul2_rn(p0, g2);
                        p1 = __fmul2_rn(p1, g2);
                    }
                    if (CAP) {   // keep p (1 - tanh^2)
                        const float2 n0 = __fmul2_rn(__fmul2_rn(s[2 * i], s[2 * i]), slope2);
                        const float2 n1 = __fmul2_rn(__fmul2_rn(s[2 * i + 1], s[2 * i + 1]), slope2);
                        s[2 * i] = __ffma2_rn(p0, n0, p0);
                        s[2 * i + 1] = __ffma2_rn(p1, n1, p1);
                    } else {
                        s[2 * i] = p0;
                        s[2 * i + 1] = p1;
                    }
                }
                tc::store16(at_s, w);
                tc::wait_st();
                tc::fence_before();
                mbar_arrive(&bars.p_ready[it & 1]);

                alive = __all_sync(0xffffffffu, wait(&bars.dp_full, it & 1));
                if (!alive) break;
                tc::fence_after();
                float2 d[16];
                tc::load32(at_dp, reinterpret_cast<float*>(d));
                tc::wait_ld();
                uint32_t rest[16];
                const float4* d4 = reinterpret_cast<const float4*>(rows[st][2] + 32 * part);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float4 dl = d4[i];
                    float2 a0 = __fadd2_rn(d[2 * i], make_float2(dl.x, dl.y));
                    float2 a1 = __fadd2_rn(d[2 * i + 1], make_float2(dl.z, dl.w));
                    a0 = __fmul2_rn(a0, s[2 * i]);
                    a1 = __fmul2_rn(a1, s[2 * i + 1]);
                    if (!whole) {   // (a hidden pair's dP need not be finite)
                        if (!(seen >> (4 * i) & 1)) a0.x = 0.f;
                        if (!(seen >> (4 * i + 1) & 1)) a0.y = 0.f;
                        if (!(seen >> (4 * i + 2) & 1)) a1.x = 0.f;
                        if (!(seen >> (4 * i + 3) & 1)) a1.y = 0.f;
                    }
                    w[2 * i] = tc::pack2<T>(a0.x, a0.y);
                    w[2 * i + 1] = tc::pack2<T>(a1.x, a1.y);
                    rest[2 * i] = tc::rest2<T>(a0, w[2 * i]);
                    rest[2 * i + 1] = tc::rest2<T>(a1, w[2 * i + 1]);
                }
                tc::store16(at_dp, w);
                tc::store16(at_dp + 16, rest);
                tc::wait_st();
                tc::fence_before();
                mbar_arrive(&bars.ds_ready[it & 1]);
            }
        }
        if (alive && total > 0) alive = __all_sync(0xffffffffu, wait(&bars.done, 0));
        const bool half = part & 1;   // even parts: dV, odd: dK, each every other 32 columns
        const uint32_t src = (half ? t_dk : t_dv) + lane_base;
        const float back = kBf16 ? 1.f : 1.f / 64.f;
        const float mul = half ? static_cast<float>(p.scale) * back * g : back;
        T* dst = static_cast<T*>(half ? gr.dk : gr.dv) +
                 ((static_cast<int64_t>(b) * p.Lk + key) * p.Hkv + hk) * p.D;
        tc::fence_after();
        if (split == 1) {
#pragma unroll 1
            for (int c = 32 * (part >> 1); c < cols; c += 64) {
                float o[32];
                if (total > 0 && alive) {
                    tc::load32(src + c, o);
                    tc::wait_ld();
                }
                if (key >= p.Lk) continue;
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    if (c + i >= p.D) break;
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w[e] = total > 0 && hi > lo
                                   ? tc::pack2<T>(o[i + 2 * e] * mul, o[i + 2 * e + 1] * mul)
                                   : 0u;
                    *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        } else {
            // this block's sums to its own shared memory, [dV, dK][column][row]
            float* own = reinterpret_cast<float*>(smem) + (half ? DP * kRows : 0);
#pragma unroll 1
            for (int c = 32 * (part >> 1); c < cols; c += 64) {
                float o[32];
                if (total > 0 && alive) {
                    tc::load32(src + c, o);
                    tc::wait_ld();
                }
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    own[(c + i) * kRows + (threadIdx.x & 127)] = total > 0 && hi > lo ? o[i] * mul : 0.f;
            }
        }
        tc::fence_before();
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 16 && lane == 0 && total > 0) {
            bool alive = true;
            mbar_arrive_expect_tx(&bars.fixed, 2 * S::tile);
            load_rows<DP>(Ks, &mk, &bars.fixed, hk, k0, b);
            load_rows<DP>(Vs, &mv, &bars.fixed, hk, k0, b);
            int it = 0, h = head0, j = fb;
            for (; it < total; ++it, ++j) {
                const int s = it % NS;
                if (j == lb) { j = fb; ++h; }
                if (it >= NS) alive = wait(&bars.empty[s], (it / NS - 1) & 1);
                if (!alive) break;
                mbar_arrive_expect_tx(&bars.x_full[s], S::tile);
                if (it == bnd.skip) { ++it; break; }
                load_rows<DP>(Q_at(s), &mq, &bars.x_full[s], h, j * kRows, b);
                mbar_arrive_expect_tx(&bars.y_full[s], S::tile);
                load_rows<DP>(O_at(s), &mo, &bars.y_full[s], h, j * kRows, b);
            }
            mbar_wait32(smem_u32(&bars.fixed), 0, bnd.timeouts);
            for (int i = max(0, it - NS); i < it; ++i)
                if (i != bnd.skip) {
                    mbar_wait32(smem_u32(&bars.x_full[i % NS]), (i / NS) & 1, bnd.timeouts);
                    mbar_wait32(smem_u32(&bars.y_full[i % NS]), (i / NS) & 1, bnd.timeouts);
                }
        } else if (warp == 17 && total > 0) {   // S and dP
            const uint32_t iss = tc::product(kBf16, 128, 128, false, false);
            const bool lead = tc::elect();
            bool fine = wait(&bars.fixed, 0);
            for (int i = 0; i < total; ++i) {
                const int s = i % NS, last = kTwoS ? i - 2 : i - 1;
                // S(i) into its place, once the product that read P there is done
                fine &= wait(&bars.x_full[s], (i / NS) & 1) && wait(&bars.ok[s], (i / NS) & 1);
                if (last >= 0) fine &= wait(&bars.used_p[last & 1], (last >> 1) & 1);
                tc::fence_after();
                if (lead) {
                    scores_mma<DP>(t_s + (kTwoS ? 128 * (i & 1) : 0), smem_u32(Ks), smem_u32(Q_at(s)),
                                   iss, steps);
                    tc::commit(smem_u32(&bars.s_full[i & 1]));
                }
                fine &= wait(&bars.y_full[s], (i / NS) & 1);
                if (i > 0) fine &= wait(&bars.used_ds[(i - 1) & 1], ((i - 1) >> 1) & 1);
                tc::fence_after();
                if (lead) {
                    scores_mma<DP>(t_dp, smem_u32(Vs), smem_u32(O_at(s)), iss, steps);
                    tc::commit(smem_u32(&bars.dp_full));
                }
                if (!__all_sync(0xffffffffu, fine)) break;
            }
            if (!__all_sync(0xffffffffu, fine)) {   // the products in flight read this block's memory
                if (lead) tc::commit(smem_u32(&bars.drain[0]));
                mbar_wait32(smem_u32(&bars.drain[0]), 0, bnd.timeouts);
            }
        } else if (warp == 18 && total > 0) {   // dV and dK
            const uint32_t its = tc::product(kBf16, 128, cols, false, true);
            const bool lead = tc::elect();
            bool fine = true;
            for (int i = 0; i < total; ++i) {
                const int s = i % NS;
                // (dO has its own barrier: P is ready as soon as Q was there.  What refills
                // the stage waits for this warp's commit, so the phase cannot pass by)
                fine &= wait(&bars.y_full[s], (i / NS) & 1);
                fine &= wait(&bars.p_ready[i & 1], (i >> 1) & 1);
                tc::fence_after();
                if (lead) {
                    mix_mma<8, 2, 32>(t_dv, t_s + (kTwoS ? 128 * (i & 1) : 0), smem_u32(O_at(s)), kPanel,
                                      its, i > 0);
                    tc::commit(smem_u32(&bars.used_p[i & 1]));
                }
                fine &= wait(&bars.ds_ready[i & 1], (i >> 1) & 1);
                tc::fence_after();
                if (lead) {
                    mix_mma<8, 2, 32>(t_dk, t_dp, smem_u32(Q_at(s)), kPanel, its, i > 0);
                    mix_mma<8, 2, 32>(t_dk, t_dp + 16, smem_u32(Q_at(s)), kPanel, its, true);
                    tc::commit(smem_u32(&bars.used_ds[i & 1]));
                    tc::commit(smem_u32(&bars.empty[s]));
                }
                if (!__all_sync(0xffffffffu, fine)) break;
            }
            if (lead) tc::commit(smem_u32(&bars.done));
            if (!__all_sync(0xffffffffu, fine)) {   // the products in flight read this block's memory
                if (lead) tc::commit(smem_u32(&bars.drain[1]));
                mbar_wait32(smem_u32(&bars.drain[1]), 0, bnd.timeouts);
            }
        } else if (warp == 19 && total > 0) {
            int h = head0, j = fb;
            for (int it = 0; it < total; ++it, ++j) {
                const int s = it % NS;
                if (j == lb) { j = fb; ++h; }
                const uint32_t parity = (it / NS) & 1;
                const RowRec* src = recs + (static_cast<int64_t>(b) * p.Hq + h) * p.Lq;
                float4 rec[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = j * kRows + lane + 32 * r;
                    rec[r] = row < p.Lq ? __ldg(reinterpret_cast<const float4*>(src + row))
                                        : make_float4(-INFINITY, 0.f, 0.f, 0.f);
                }
                if (it >= NS && !wait(&bars.empty[s], parity ^ 1)) break;
                uint32_t bad = 0;
                if (guarded(j)) {
                    if (!wait(&bars.x_full[s], parity) || !wait(&bars.y_full[s], parity)) break;
                    bad = scrub_rows<T, DP>(Q_at(s), lane, 32) | scrub_rows<T, DP>(O_at(s), lane, 32);
                    fence_async_shared();
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at = lane + 32 * r;
                    float m = -rec[r].x, ll = -rec[r].y + (kBf16 ? 0.f : kPShift);
                    if (rec[r].x == -INFINITY) m = -INFINITY;   // sees nothing: weight zero
                    if (bad >> r & 1) m = NAN;
                    rows[s][0][at] = BIAS ? m : m + ll;
                    rows[s][1][at] = ll;
                    rows[s][2][at] = -rec[r].z;
                }
                mbar_arrive(&bars.ok[s]);
            }
        }
        __syncwarp();
    }
    if (split > 1) {
        // Joined over the cluster in the order of its ranks: block `rank` sums its share of
        // the columns, four at a time, from every block's shared memory.
        cluster_sync();
        if (warp < 16 && k0 + static_cast<int>(threadIdx.x & 127) < p.Lk) {
            const int row = threadIdx.x & 127, groups = cols / 4;
            for (int x = static_cast<int>(threadIdx.x >> 7) * split + rank; x < 2 * groups;
                 x += 4 * split) {
                const bool half = x >= groups;
                const int c = (half ? x - groups : x) * 4;
                if (c >= p.D) continue;
                const uint32_t at = smem_u32(reinterpret_cast<float*>(smem) +
                                             ((half ? DP : 0) + c) * kRows + row);
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
                for (int r = 0; r < split; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[e] += cluster_load<float>(at + e * kRows * 4, r);
                T* dst = static_cast<T*>(half ? gr.dk : gr.dv) +
                         ((static_cast<int64_t>(b) * p.Lk + k0 + row) * p.Hkv + hk) * p.D + c;
                *reinterpret_cast<uint2*>(dst) =
                    make_uint2(tc::pack2<T>(sum[0], sum[1]), tc::pack2<T>(sum[2], sum[3]));
            }
        }
        cluster_sync();   // no block leaves while another reads its memory
    }
    __syncthreads();
    if (warp == 17) {
        tc::fence_after();
        tc::tmem_free(tmem, 512);
    }
}

template <typename T, int DP, bool CAP, bool BIAS>
__global__ __launch_bounds__(kBwdThreads, 1) void tc_dq_kernel(
    const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mo,
    const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const Params p,
    const Grads gr, const RowRec* __restrict__ recs, const Bounded bnd) {
    using S = BwdShape<DP>;
    constexpr int NS = S::stages;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ unsigned char smem_raw[];
    __shared__ BwdBars bars;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag[2];
    __shared__ int span[4];
    __shared__ float diag[16][64], far_sum[16][2];
    unsigned char* smem = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    unsigned char* Qs = smem;
    unsigned char* Os = smem + S::tile;
    unsigned char* ring = smem + 2 * S::tile;   // stages of K, V
    float* E = reinterpret_cast<float*>(smem + S::smem);
    float* acc = E + 2 * p.reach + 2 * kBiasPad + 1;   // table sums, 16 warps by buckets

    const int warp = tc::uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    const int64_t BH = static_cast<int64_t>(p.B) * p.Hq;
    const int nt = (p.Lq + kRows - 1) / kRows;
    const int t = nt - 1 - static_cast<int>(blockIdx.x / BH);
    const int bh = static_cast<int>(blockIdx.x % BH), b = bh / p.Hq, h = bh % p.Hq;
    const int hk = h / p.G, q0 = t * kRows, off = p.Lk - p.Lq;

    if (threadIdx.x < 4) span[threadIdx.x] = threadIdx.x == 0 || threadIdx.x == 3 ? INT_MAX : 0;
    if (threadIdx.x == 0) {
        mbar_init(&bars.fixed, 1);
        for (int i = 0; i < NS; ++i) {
            mbar_init(&bars.x_full[i], 1);
            mbar_init(&bars.y_full[i], 1);
            mbar_init(&bars.empty[i], 1);
            mbar_init(&bars.ok[i], 32);
        }
        mbar_init(&bars.ds_ready[0], kBwdMath);
        mbar_init(&bars.ds_ready[1], kBwdMath);
        mbar_init(&bars.dp_full, 1);
        mbar_init(&bars.dp_free, kBwdMath);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.used_p[i], 1);
            mbar_init(&bars.used_ds[i], 1);
        }
        mbar_init(&bars.done, 1);
        mbar_init(&bars.drain[0], 1);
        mbar_init(&bars.drain[1], 1);
        fence_mbar_init();
        abort_flag[0] = 0;
        abort_flag[1] = static_cast<int>(bnd.budget);
    }
    if (warp == 17) tc::tmem_alloc(&tmem_slot, 512);
    if (BIAS) {
        load_padded_bias(p, h, E, threadIdx.x, kBwdThreads);
        if (gr.tab)
            for (int i = threadIdx.x; i < 16 * p.nb; i += kBwdThreads) acc[i] = 0.f;
    }
    __syncthreads();
    const int row = q0 + static_cast<int>(threadIdx.x & 127);
    int lo = 0, hi = 0;
    if (warp < 16) {
        if (row < p.Lq) key_span(p, b, row, p.Lk, lo, hi);
        const int v0 = __reduce_min_sync(0xffffffffu, hi > lo ? lo : INT_MAX);
        const int v1 = __reduce_max_sync(0xffffffffu, hi > lo ? hi : 0);
        const int v2 = __reduce_max_sync(0xffffffffu, hi > lo ? lo : 0);
        const int v3 = __reduce_min_sync(0xffffffffu, hi > lo ? hi : INT_MAX);
        if (lane == 0 && warp < 4) {
            atomicMin(&span[0], v0);
            atomicMax(&span[1], v1);
            atomicMax(&span[2], v2);
            atomicMin(&span[3], v3);
        }
    }
    __syncthreads();
    const uint32_t tmem = tc::uniform(tmem_slot);
    const int s_lo = tc::uniform(span[0]), s_hi = tc::uniform(span[1]);
    const int all_lo = tc::uniform(span[2]), all_hi = tc::uniform(span[3]);
    const int fb = s_hi > s_lo ? s_lo / kRows : 0;
    const int lb = s_hi > s_lo ? (s_hi + kRows - 1) / kRows : 0;
    const int total = lb - fb;
    auto guarded = [&](int j) {
        return !(j * kRows >= all_lo && min((j + 1) * kRows, p.Lk) <= all_hi);
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        return wait_bounded(bar, parity, bnd.timeouts, abort_flag);
    };
    auto K_at = [&](int s) { return ring + s * 2 * S::tile; };
    auto V_at = [&](int s) { return ring + s * 2 * S::tile + S::tile; };
    const int steps = (p.D + 15) / 16, cols = steps * 16;
    const uint32_t t_s = tmem, t_dp = tmem + 256, t_dq = tmem + 384;

    if (warp < 16) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMathRegs));
        const int part = warp >> 2;
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t at_s = t_s + lane_base + 32 * part, at_dp = t_dp + lane_base + 32 * part;
        const float unit = static_cast<float>((p.cap > 0 ? p.cap : p.scale) * kLog2e);
        const float y1 = p.cap > 0 ? static_cast<float>(p.scale / p.cap) : 0.f;
        float m = -INFINITY, ll = 0.f, delta = 0.f, norm = 0.f, g = 1.f;
        // (a row that sees nothing keeps its zeros, whatever its output gradient holds)
        if (hi > lo) {
            const float4 r = __ldg(reinterpret_cast<const float4*>(
                recs + (static_cast<int64_t>(b) * p.Hq + h) * p.Lq + row));
            m = r.x == -INFINITY ? r.x : -r.x;
            ll = -r.y + (kBf16 ? 0.f : kPShift);
            delta = -r.z;
            norm = r.w;
        }
        if (!kBf16 && hi > lo) {
            g = gradient_scale(norm * __ldg(gr.seen_norms + (static_cast<int64_t>(b) * p.Hkv + hk) * p.Lq + row) +
                               fabsf(delta));
            delta /= g;
        }
        if (!BIAS) m += ll;
        const Cap<T> cap(y1, unit);
        const float2 u2 = CAP ? make_float2(1.f, 1.f) : make_float2(unit, unit);
        const float2 g2 = make_float2(1.f / g, 1.f / g);
        const float2 slope2 = make_float2(-1.f / (unit * unit), -1.f / (unit * unit));   // 1 - tanh^2 = 1 + s^2 slope
        const float2 m2 = make_float2(m, m), l2 = make_float2(ll, ll), d2 = make_float2(delta, delta);
        // (a row whose output gradient is not finite has m NaN: its hidden pairs are
        // taken out of the table's sums one by one)
        const bool odd_row = BIAS && !CAP && __any_sync(0xffffffffu, m != m);
        float far_lo = 0.f, far_hi = 0.f;
        const float undo = kBf16 ? 1.f : g / 64.f;
        bool alive = true;
        int it = 0;
        for (int j = fb; j < lb; ++j, ++it) {
            alive = __all_sync(0xffffffffu, wait(&bars.dp_full, it & 1));
            if (!alive) break;
            tc::fence_after();
            float2 s[16], d[16];
            const uint32_t as = at_s + 128 * (it & 1);
            tc::load32(at_dp, reinterpret_cast<float*>(d));
            tc::load32(as, reinterpret_cast<float*>(s));
            tc::wait_ld();
            tc::fence_before();
            mbar_arrive(&bars.dp_free);
            if (CAP) cap(s);
            const int k0 = j * kRows + 32 * part;
            const bool whole = __all_sync(0xffffffffu, lo <= k0 && hi >= k0 + 32);
            const uint32_t seen = whole ? 0 : seen_bits(lo - k0, hi - k0);
            // out of the loop where it can be: P = 2^-inf and dP = 0 give dS = 0 (a capped
            // score would give 0 x inf by its slope)
            if (!CAP && !whole) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (!(seen >> (2 * i) & 1)) s[i].x = -INFINITY, d[i].x = 0.f;
                    if (!(seen >> (2 * i + 1) & 1)) s[i].y = -INFINITY, d[i].y = 0.f;
                }
            }
            const int rel0 = k0 - (row + off);   // distance at column 0, one more a column
            const int w0 = __shfl_sync(0xffffffffu, rel0, 0);   // lane r: w0 - r
            bool far = false;
            float e_far = 0.f;
            if (BIAS) {
                far = w0 + 31 <= -p.reach || w0 - 31 >= p.reach;
                if (far) e_far = E[w0 > 0 ? 2 * p.reach + kBiasPad : kBiasPad];
            }
            const float* er = E + rel0 + p.reach + kBiasPad;
            uint32_t w[16], rest[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float2 x;
                if (BIAS) {
                    float2 e = make_float2(e_far, e_far);
                    if (!far) e = make_float2(er[2 * i], er[2 * i + 1]);
                    x = __fadd2_rn(__fadd2_rn(__ffma2_rn(s[i], u2, e), m2), l2);
                } else {
                    x = __ffma2_rn(s[i], u2, m2);
                }
                const float2 pr = make_float2(tc::ex2(x.x), tc::ex2(x.y));
                float2 z = kBf16 ? __fadd2_rn(d[i], d2) : __ffma2_rn(d[i], g2, d2);
                z = __fmul2_rn(z, pr);
                if (CAP && !whole) {
                    if (!(seen >> (2 * i) & 1)) z.x = 0.f;
                    if (!(seen >> (2 * i + 1) & 1)) z.y = 0.f;
                }
                if (BIAS) d[i] = z;
                if (CAP) {
                    const float2 n = __fmul2_rn(__fmul2_rn(s[i], s[i]), slope2);
                    z = __ffma2_rn(z, n, z);
                }
                w[i] = tc::pack2<T>(z.x, z.y);
                rest[i] = tc::rest2<T>(z, w[i]);
            }
            tc::store16(as, w);
            tc::store16(as + 16, rest);
            tc::wait_st();
            tc::fence_before();
            mbar_arrive(&bars.ds_ready[it & 1]);
            if (BIAS && gr.tab) {
                if (!CAP && odd_row && !whole) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if (!(seen >> (2 * i) & 1)) d[i].x = 0.f;
                        if (!(seen >> (2 * i + 1) & 1)) d[i].y = 0.f;
                    }
                }
                if (far) {
                    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum = __fadd2_rn(sum, d[i]);
                    const float v = (sum.x + sum.y) * undo;
                    if (w0 > 0) far_hi += v; else far_lo += v;
                } else {
                    // sums along the diagonals of the warp's 32 x 32 part: a sum moves
                    // one lane up a column, and is whole in lane 31, or where it is at
                    // the end.  Entry 31 + c - r.
                    float a = 0.f;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float z = (i & 1) ? d[i >> 1].y : d[i >> 1].x;
                        a = __shfl_up_sync(0xffffffffu, a, 1);
                        a = fmaf(z, undo, lane == 0 ? 0.f : a);
                        if (lane == 31) diag[warp][i] = a;
                    }
                    if (lane < 31) diag[warp][62 - lane] = a;
                    __syncwarp();
                    for (int u = lane; u < p.nb; u += 32) {
                        float sum = 0.f;
                        for (int i = 0; i < 63; ++i) {
                            const int at = min(max(w0 + i - 31, -p.reach), p.reach) + p.reach;
                            const int bu = min(max(__ldg(p.lut + at), 0), p.nb - 1);
                            if (bu == u) sum += diag[warp][i];
                        }
                        acc[warp * p.nb + u] += sum;
                    }
                    __syncwarp();
                }
            }
        }
        if (BIAS && gr.tab) {
#pragma unroll
            for (int i = 16; i; i >>= 1) {
                far_lo += __shfl_xor_sync(0xffffffffu, far_lo, i);
                far_hi += __shfl_xor_sync(0xffffffffu, far_hi, i);
            }
            if (lane == 0) {
                far_sum[warp][0] = far_lo;
                far_sum[warp][1] = far_hi;
            }
        }
        if (alive && total > 0) alive = __all_sync(0xffffffffu, wait(&bars.done, 0));
        if (alive) {
            tc::fence_after();
            const float mul = static_cast<float>(p.scale) * undo;
            T* dst = static_cast<T*>(gr.dq) +
                     ((static_cast<int64_t>(b) * p.Lq + row) * p.Hq + h) * p.D;
#pragma unroll 1
            for (int c = 32 * part; c < cols; c += 128) {
                float o[32];
                if (total > 0) {
                    tc::load32(t_dq + lane_base + c, o);
                    tc::wait_ld();
                }
                if (row >= p.Lq) continue;
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    if (c + i >= p.D) break;
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w[e] = total > 0 && hi > lo
                                   ? tc::pack2<T>(o[i + 2 * e] * mul, o[i + 2 * e + 1] * mul)
                                   : 0u;
                    *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            tc::fence_before();
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 16 && lane == 0 && total > 0) {
            bool alive = true;
            mbar_arrive_expect_tx(&bars.fixed, 2 * S::tile);
            load_rows<DP>(Qs, &mq, &bars.fixed, h, q0, b);
            load_rows<DP>(Os, &mo, &bars.fixed, h, q0, b);
            int it = 0;
            for (; it < total; ++it) {
                const int s = it % NS, j = fb + it;
                if (it >= NS) alive = wait(&bars.empty[s], (it / NS - 1) & 1);
                if (!alive) break;
                mbar_arrive_expect_tx(&bars.x_full[s], S::tile);
                if (it == bnd.skip) { ++it; break; }
                load_rows<DP>(K_at(s), &mk, &bars.x_full[s], hk, j * kRows, b);
                mbar_arrive_expect_tx(&bars.y_full[s], S::tile);
                load_rows<DP>(V_at(s), &mv, &bars.y_full[s], hk, j * kRows, b);
            }
            mbar_wait32(smem_u32(&bars.fixed), 0, bnd.timeouts);
            for (int i = max(0, it - NS); i < it; ++i)
                if (i != bnd.skip) {
                    mbar_wait32(smem_u32(&bars.x_full[i % NS]), (i / NS) & 1, bnd.timeouts);
                    mbar_wait32(smem_u32(&bars.y_full[i % NS]), (i / NS) & 1, bnd.timeouts);
                }
        } else if (warp == 17 && total > 0) {   // S and dP
            const uint32_t iss = tc::product(kBf16, 128, 128, false, false);
            const bool lead = tc::elect();
            bool fine = wait(&bars.fixed, 0);
            for (int i = 0; i < total; ++i) {
                const int s = i % NS;
                fine &= wait(&bars.x_full[s], (i / NS) & 1) && wait(&bars.ok[s], (i / NS) & 1);
                // (the place of S(i) holds dS of the block before last until dQ has read it)
                if (i > 1) fine &= wait(&bars.used_ds[i & 1], ((i - 2) >> 1) & 1);
                tc::fence_after();
                if (lead)
                    scores_mma<DP>(t_s + 128 * (i & 1), smem_u32(Qs), smem_u32(K_at(s)), iss, steps);
                fine &= wait(&bars.y_full[s], (i / NS) & 1);
                if (i > 0) fine &= wait(&bars.dp_free, (i - 1) & 1);
                tc::fence_after();
                if (lead) {
                    scores_mma<DP>(t_dp, smem_u32(Os), smem_u32(V_at(s)), iss, steps);
                    tc::commit(smem_u32(&bars.dp_full));
                }
                if (!__all_sync(0xffffffffu, fine)) break;
            }
            if (!__all_sync(0xffffffffu, fine)) {   // the products in flight read this block's memory
                if (lead) tc::commit(smem_u32(&bars.drain[0]));
                mbar_wait32(smem_u32(&bars.drain[0]), 0, bnd.timeouts);
            }
        } else if (warp == 18 && total > 0) {   // dQ
            const uint32_t its = tc::product(kBf16, 128, cols, false, true);
            const bool lead = tc::elect();
            bool fine = true;
            for (int i = 0; i < total; ++i) {
                const int s = i % NS;
                fine &= wait(&bars.ds_ready[i & 1], (i >> 1) & 1);
                tc::fence_after();
                if (lead) {
                    const uint32_t w = t_s + 128 * (i & 1);
                    mix_mma<8, 2, 32>(t_dq, w, smem_u32(K_at(s)), kPanel, its, i > 0);
                    mix_mma<8, 2, 32>(t_dq, w + 16, smem_u32(K_at(s)), kPanel, its, true);
                    tc::commit(smem_u32(&bars.used_ds[i & 1]));
                    tc::commit(smem_u32(&bars.empty[s]));
                }
                if (!__all_sync(0xffffffffu, fine)) break;
            }
            if (lead) tc::commit(smem_u32(&bars.done));
            if (!__all_sync(0xffffffffu, fine)) {   // the products in flight read this block's memory
                if (lead) tc::commit(smem_u32(&bars.drain[1]));
                mbar_wait32(smem_u32(&bars.drain[1]), 0, bnd.timeouts);
            }
        } else if (warp == 19 && total > 0) {
            for (int it = 0; it < total; ++it) {
                const int s = it % NS;
                const uint32_t parity = (it / NS) & 1;
                if (it >= NS && !wait(&bars.empty[s], parity ^ 1)) break;
                if (guarded(fb + it)) {
                    if (!wait(&bars.x_full[s], parity) || !wait(&bars.y_full[s], parity)) break;
                    const uint32_t bad = scrub_rows<T, DP>(K_at(s), lane, 32);
#pragma unroll
                    for (int r = 0; r < 4; ++r)   // the rows that see it get NaN by dP
                        if (bad >> r & 1) poison_row<DP>(V_at(s), lane + 32 * r);
                    fence_async_shared();
                }
                mbar_arrive(&bars.ok[s]);
            }
        }
        __syncwarp();
    }
    __syncthreads();
    if (BIAS && gr.tab && static_cast<int>(threadIdx.x) < p.nb) {
        const int u = threadIdx.x;
        const int b_lo = min(max(__ldg(p.lut), 0), p.nb - 1);
        const int b_hi = min(max(__ldg(p.lut + 2 * p.reach), 0), p.nb - 1);
        float sum = 0.f;
        for (int i = 0; i < 16; ++i) {
            sum += acc[i * p.nb + u];
            if (u == b_lo) sum += far_sum[i][0];
            if (u == b_hi) sum += far_sum[i][1];
        }
        static_cast<float*>(gr.tab)[(static_cast<int64_t>(h) * gr.n_part + b * nt + t) * p.nb + u] = sum;
    }
    if (warp == 17) {
        tc::fence_after();
        tc::tmem_free(tmem, 512);
    }
}

template <typename T, int DP, bool CAP, bool BIAS>
nsc_status tc_bwd_launch(const Params& p, const Grads& g, const RowRec* recs, cudaStream_t st) {
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    auto kk = tc_dkv_kernel<T, DP, CAP, BIAS>;
    auto kq = tc_dq_kernel<T, DP, CAP, BIAS>;
    const int e = BIAS ? 4 * (2 * p.reach + 2 * kBiasPad + 1) : 0;
    const int smk = BwdShape<DP>::smem + 1024 + e;
    const int smq = smk + (BIAS && g.tab ? 4 * 16 * p.nb : 0);
    const int regs = kBwdMath * kMathRegs + 128 * kOtherRegs;
    const char* op = "token_attention backward";
    nsc_status ready = raise_shared(op, reinterpret_cast<const void*>(kk), smk, kBwdThreads, regs);
    if (ready == NSC_OK)
        ready = raise_shared(op, reinterpret_cast<const void*>(kq), smq, kBwdThreads, regs);
    if (ready != NSC_OK) return ready;
    CUtensorMap mq, mo, mk, mv;
    const char* err = nullptr;
    if (!encode_heads(&mq, p.q, p.qs, p.B, p.Lq, p.Hq, p.D, kBf16, &err) ||
        !encode_heads(&mo, g.dout, g.dos, p.B, p.Lq, p.Hq, p.D, kBf16, &err) ||
        !encode_heads(&mk, p.k, p.ks, p.B, p.Lk, p.Hkv, p.D, kBf16, &err) ||
        !encode_heads(&mv, p.v, p.vs, p.B, p.Lk, p.Hkv, p.D, kBf16, &err))
        return fail(NSC_ERR_LAUNCH_FAILED, "token_attention backward: %s", err);
    Bounded bnd{wait_timeout_counter(), -1, 0};
    if (!bnd.timeouts)
        return fail(NSC_ERR_LAUNCH_FAILED, "token_attention backward: no wait counter");
    wait_fault_settings(&bnd.skip, &bnd.budget);
    // Blocks of a cluster share the query heads of a key head where there would be fewer
    // than three blocks an SM: the few long blocks of a causal or packed batch end last.
    // No more of them than that takes, since a cluster's blocks have to find SMs side by
    // side.  (16 heads on 4, four documents in 8192 tokens, 256 key tiles of 4 heads: 500 us
    // alone, 341 in twos, 402 in fours.)
    const int64_t tiles = static_cast<int64_t>((p.Lk + kRows - 1) / kRows) * p.B * p.Hkv;
    int split = 1;
    for (int i = 2; i <= 8 && tiles * split < 3 * 148; ++i)
        if (p.G % i == 0) split = i;
    const int64_t nk = tiles * split;
    const int64_t nq = static_cast<int64_t>((p.Lq + kRows - 1) / kRows) * p.B * p.Hq;
    if (g.dk)
        ready = launch_cluster("token_attention backward", kk, nk, kBwdThreads, smk, split, st, mq, mo, mk,
                           mv, p, g, recs, split, bnd);
    if (ready != NSC_OK || !g.dq) return ready;
    kq<<<static_cast<unsigned>(nq), kBwdThreads, smq, st>>>(mq, mo, mk, mv, p, g, recs, bnd);
    return check_launch("token_attention backward");
}

}  // namespace

template <typename T, int DP>
nsc_status tc_bwd_run(const Params& p, const Grads& g, const void* recs, cudaStream_t st) {
    const RowRec* r = static_cast<const RowRec*>(recs);
    if (p.cap > 0)
        return p.table ? tc_bwd_launch<T, DP, true, true>(p, g, r, st)
                       : tc_bwd_launch<T, DP, true, false>(p, g, r, st);
    return p.table ? tc_bwd_launch<T, DP, false, true>(p, g, r, st)
                   : tc_bwd_launch<T, DP, false, false>(p, g, r, st);
}

}  // namespace tok
}  // namespace nsc
