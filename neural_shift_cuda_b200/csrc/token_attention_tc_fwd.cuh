// token_attention_tc_fwd.cuh -- forward of token attention on the tensor
// cores, fp16 / bf16, head widths up to 128.
//
// A block owns a tile of 128 queries of a head; two blocks share an SM, so that one's
// set-up and output (some 5 us of a block's time) pass beside the other's products, and
// each fills the other's waits.  (One block of two tiles an SM: 16 heads of 128, 8192 keys
// 521 against 470 us; 16 heads of 64, 8191 packed tokens 107 against 96, since 92.)  Roles by warp:
// 0-3 the softmax, a thread a row; 4 loads K and V blocks of 64 keys through a ring by
// TMA; 5 issues the products; 7 guards (below).
//
// Tensor memory holds O and two S: S(j+1) is computed beside the softmax of block j.
// P takes the place of its S as 16-bit pairs.  (Products of different shapes or
// accumulators need not complete in the order of their issue: whatever overwrites an
// operand waits for its reader's commit.)  Keys are released after their scores and values
// after PV: heads of 128 have room for two stages only, and released together the
// next keys came too late (669 against 470 us).
//
// Softmax with a running reference m: p = 2^(s2 - m); m moves, and O is
// rescaled, only when a row's maximum passes m + 8 (p <= 256 keeps 16-bit
// weights in range), which after the first blocks is rare.  P is rounded to the
// operand type; the sum of a row is of the fp32 values.  REST, for training
// (a residue is wanted): what that rounding drops is multiplied too, as a second operand.
// The backward's row sums of grad_out * out are then those of the weights it recomputes;
// without it the score gradients of rows with few keys, and the sums of many such terms in
// a bucket, lose digits (documents of some keys, bf16: grad_q and grad_k 2.8e-3 off
// instead of 1.7e-3, which is their own rounding; a bucket of 8192 rows 3.1e-3 instead of
// 1.7e-3).  It costs some 15 % of a capped forward with heads of 128 (200 -> 230 us when
// it came, 16 heads, 8192 tokens in 4 documents).
//
// Guard: in blocks that some row of a tile does not see whole, a value row
// that is not finite would reach every row as 0 x NaN.  There the guard warp
// looks each landed V block over; such a row becomes zero in V and NaN in K,
// so that the rows that see it still give NaN, by their scores.
//
// 8192 keys, 16 heads, bf16: 470 us with heads of 128 (1170 TF/s, 0.71 of a library
// product's rate), 413 us with heads of 64 (665 TF/s).  Work per score: one exponential
// (16 a clock and SM) against D / 32 tensor-core clocks; heads of 64 are bounded by the
// softmax's latency at two warps a scheduler (exponential unit half busy), heads of 128
// by that and the products about alike, capped scores by the FMA pipe too.
#pragma once

#include "token_attention_tc.cuh"

namespace nsc {
namespace tok {
namespace {

constexpr int kFwdThreads = 256, kFwdMathRegs = 176, kFwdOtherRegs = 80;
constexpr float kLazy = 8.f;

constexpr int kKeys = 64;   // keys of a block

template <int DP> struct FwdShape {
    static constexpr int tile = DP / 64 * kPanel;                  // bytes of a query tile
    static constexpr int panel = kKeys * 128, block = DP / 64 * panel;   // of a K or V block
    static constexpr int stages = DP == 64 ? 5 : 2;                // K and V blocks in flight
    static constexpr int smem = tile + stages * 2 * block;         // + bias + 1024 of alignment
};

struct FwdBars {
    // (two of s_full and p_full, for even and odd blocks: the products, and a fast warp,
    // may be a block ahead of a slow warp)
    uint64_t q, k_full[5], v_full[5], k_empty[5], v_empty[5], ok[5], s_full[2], p_full[2], pv, o_full, drain;
};

template <typename T, int DP, bool CAP, bool BIAS, bool REST>
__global__ __launch_bounds__(kFwdThreads, 2) void tc_fwd_kernel(
    const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
    const __grid_constant__ CUtensorMap mv, const Params p, const Bounded bnd) {
    using S = FwdShape<DP>;
    constexpr int NS = S::stages;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ unsigned char smem_raw[];
    __shared__ FwdBars bars;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag[2];
    __shared__ int span[4];   // of the rows: least lo, most hi, most lo, least hi
    unsigned char* smem = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    unsigned char* Qs = smem;
    unsigned char* KV = smem + S::tile;             // stages of K, V
    float* E = reinterpret_cast<float*>(smem + S::smem);

    const int warp = tc::uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    const int64_t BH = static_cast<int64_t>(p.B) * p.Hq;
    const int nt = gridDim.x / BH;
    const int t = nt - 1 - static_cast<int>(blockIdx.x / BH);   // (causal: the longest first)
    const int bh = static_cast<int>(blockIdx.x % BH), b = bh / p.Hq, h = bh % p.Hq;
    const int hk = h / p.G, n = keys_of(p, b);
    const int q0 = t * kRows;

    if (threadIdx.x < 4) span[threadIdx.x] = threadIdx.x == 0 || threadIdx.x == 3 ? INT_MAX : 0;
    if (threadIdx.x == 0) {
        mbar_init(&bars.q, 1);
        for (int i = 0; i < NS; ++i) {
            mbar_init(&bars.k_full[i], 1);
            mbar_init(&bars.v_full[i], 1);
            mbar_init(&bars.k_empty[i], 1);
            mbar_init(&bars.v_empty[i], 1);
            mbar_init(&bars.ok[i], 32);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.s_full[i], 1);
            mbar_init(&bars.p_full[i], kRows);
        }
        mbar_init(&bars.pv, 1);
        mbar_init(&bars.o_full, 1);
        mbar_init(&bars.drain, 1);
        fence_mbar_init();
        abort_flag[0] = 0;
        abort_flag[1] = static_cast<int>(bnd.budget);
    }
    if (warp == 5) tc::tmem_alloc(&tmem_slot, 256);
    __syncthreads();

    // the rows' spans, and the tile's
    const int row = q0 + static_cast<int>(threadIdx.x & 127);
    int lo = 0, hi = 0;
    if (warp < 4) {
        if (row < p.Lq) key_span(p, b, row, n, lo, hi);
        int v0 = hi > lo ? lo : INT_MAX, v1 = hi > lo ? hi : 0;
        int v2 = hi > lo ? lo : 0, v3 = hi > lo ? hi : INT_MAX;
        v0 = __reduce_min_sync(0xffffffffu, v0);
        v1 = __reduce_max_sync(0xffffffffu, v1);
        v2 = __reduce_max_sync(0xffffffffu, v2);
        v3 = __reduce_min_sync(0xffffffffu, v3);
        if (lane == 0) {
            atomicMin(&span[0], v0);
            atomicMax(&span[1], v1);
            atomicMax(&span[2], v2);
            atomicMin(&span[3], v3);
        }
        // (a row past the end is not written; it must not make a block look partly seen)
        if (row >= p.Lq) hi = INT_MAX;
    }
    if (BIAS) load_padded_bias(p, h, E, threadIdx.x, kFwdThreads);
    __syncthreads();
    const uint32_t tmem = tc::uniform(tmem_slot);
    const int s0 = tc::uniform(span[0]), s1 = tc::uniform(span[1]);
    const int all_lo = tc::uniform(span[2]), all_hi = tc::uniform(span[3]);   // keys that all rows see
    const int j0 = s1 > s0 ? s0 / kKeys : 0, j1 = s1 > s0 ? (s1 + kKeys - 1) / kKeys : 0;   // key blocks
    auto guarded = [&](int j) {
        return !(j * kKeys >= all_lo && min((j + 1) * kKeys, n) <= all_hi);
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        return wait_bounded(bar, parity, bnd.timeouts, abort_flag);
    };
    auto K_at = [&](int s) { return KV + s * 2 * S::block; };
    auto V_at = [&](int s) { return KV + s * 2 * S::block + S::block; };
    const int steps = (p.D + 15) / 16;   // of 16 channels
    const int cols = steps * 16;

    if (warp < 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFwdMathRegs));
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t to = tmem + 128 + lane_base;
        const int pos = row + n - p.Lq;
        const float unit = static_cast<float>((p.cap > 0 ? p.cap : p.scale) * kLog2e);
        const float y1 = p.cap > 0 ? static_cast<float>(p.scale / p.cap) : 0.f;
        const Cap<T> cap(y1, unit);
        float m = -INFINITY, l = 0.f;
        bool alive = true;
        int it = 0;
        for (int j = j0; j < j1; ++j, ++it) {
            alive = __all_sync(0xffffffffu, wait(&bars.s_full[it & 1], (it >> 1) & 1));
            if (!alive) break;
            tc::fence_after();
            const uint32_t ts = tmem + lane_base + (it & 1) * kKeys;
            float2 s[32];
            tc::load32(ts, reinterpret_cast<float*>(s));
            tc::load32(ts + 32, reinterpret_cast<float*>(s + 16));
            tc::wait_ld();
            const int k0 = j * kKeys;
            if (CAP) {
                cap(s);
                cap(s + 16);
            }
            const float mul = CAP || BIAS ? 1.f : unit;   // of what `s` holds then
            if (BIAS) {
                const int w0 = __shfl_sync(0xffffffffu, pos, 0);   // lanes at w0 .. w0 + 31
                const float2 u2 = CAP ? make_float2(1.f, 1.f) : make_float2(unit, unit);
                if (k0 + kKeys - 1 - w0 <= -p.reach || k0 - w0 - 31 >= p.reach) {
                    const float e = E[k0 > w0 ? 2 * p.reach + kBiasPad : kBiasPad];
                    const float2 e2 = make_float2(e, e);
#pragma unroll
                    for (int i = 0; i < 32; ++i) s[i] = __ffma2_rn(s[i], u2, e2);
                } else {
                    const float* er = E + (k0 - pos + p.reach + kBiasPad);
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        s[i] = __ffma2_rn(s[i], u2, make_float2(er[2 * i], er[2 * i + 1]));
                }
            }
            if (!__all_sync(0xffffffffu, lo <= k0 && hi >= k0 + kKeys)) {
                // (a bit a key: an element then costs a test of a constant bit; two compares
                // an element were 4 % of a packed call)
                const uint32_t seen[2] = {seen_bits(lo - k0, hi - k0), seen_bits(lo - k0 - 32, hi - k0 - 32)};
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    if (!(seen[i / 16] >> (2 * i % 32) & 1)) s[i].x = -INFINITY;
                    if (!(seen[i / 16] >> (2 * i % 32 + 1) & 1)) s[i].y = -INFINITY;
                }
            }
            // (four maxima, and four sums below, side by side: one chain would wait
            // out the latency of each of its 64 steps)
            float tops[4] = {s[0].x, s[1].x, s[2].x, s[3].x};
#pragma unroll
            for (int i = 0; i < 32; ++i) tops[i & 3] = fmaxf(tops[i & 3], fmaxf(s[i].x, s[i].y));
            const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * mul;
            // (a row may see nothing of its first blocks: m is then -inf still)
            float keep = 1.f;
            if (top > m + kLazy || m == -INFINITY) {
                keep = m == -INFINITY ? 0.f : tc::ex2(m - top);
                m = fmaxf(top, m);
            }
            if (it > 0 && __any_sync(0xffffffffu, keep != 1.f)) {
                // (PV of the last block is done, and this one's has not begun)
                alive = __all_sync(0xffffffffu, wait(&bars.pv, (it - 1) & 1));
                if (!alive) break;
                tc::fence_after();
                l *= keep;
                const float2 k2 = make_float2(keep, keep);
#pragma unroll 1
                for (int c = 0; c < cols; c += 16) {
                    float2 o[8];
                    tc::load16(to + c, reinterpret_cast<float*>(o));
                    tc::wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = __fmul2_rn(o[i], k2);
                    tc::store16(to + c, reinterpret_cast<uint32_t*>(o));
                }
            }
            const float ref = m == -INFINITY ? 0.f : -m;
            const float2 mul2 = make_float2(mul, mul), ref2 = make_float2(ref, ref);
            float2 sums[4] = {};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t w[16], rest[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 x = __ffma2_rn(s[16 * c + i], mul2, ref2);
                    const float2 e = make_float2(tc::ex2(x.x), tc::ex2(x.y));
                    sums[i & 3] = __fadd2_rn(sums[i & 3], e);
                    w[i] = tc::pack2<T>(e.x, e.y);
                    if (REST) rest[i] = tc::rest2<T>(e, w[i]);
                }
                tc::store16(ts + 16 * c, w);
                if (REST) tc::store16(ts + 32 + 16 * c, rest);
            }
            const float2 sum = __fadd2_rn(__fadd2_rn(sums[0], sums[1]), __fadd2_rn(sums[2], sums[3]));
            l += sum.x + sum.y;
            tc::wait_st();
            tc::fence_before();
            mbar_arrive(&bars.p_full[it & 1]);
        }
        // the row's output
        const bool worked = j1 > j0;
        if (alive && worked) alive = __all_sync(0xffffffffu, wait(&bars.o_full, 0));
        if (alive) {
            tc::fence_after();
            const bool none = l == 0.f;
            const float inv = none ? 0.f : 1.f / l;
            const int64_t at = ((static_cast<int64_t>(b) * p.Lq + row) * p.Hq + h) * p.D;
#pragma unroll 1
            for (int c = 0; c < cols; c += 32) {
                float o[32];
                if (worked) {
                    tc::load32(to + c, o);
                    tc::wait_ld();
                }
                if (row >= p.Lq) continue;
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    if (c + i >= p.D) break;
                    uint32_t w[4], r[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = none ? 0.f : o[i + 2 * e] * inv;
                        const float y = none ? 0.f : o[i + 2 * e + 1] * inv;
                        w[e] = tc::pack2<T>(x, y);
                        const T* back = reinterpret_cast<const T*>(&w[e]);
                        r[e] = tc::pack2<T>(x - to_acc(back[0]), y - to_acc(back[1]));
                    }
                    *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + at + c + i) =
                        make_uint4(w[0], w[1], w[2], w[3]);
                    if (p.residue)
                        *reinterpret_cast<uint4*>(static_cast<T*>(p.residue) + at + c + i) =
                            make_uint4(r[0], r[1], r[2], r[3]);
                }
            }
            if (row < p.Lq)
                row_stats<float>(p, (static_cast<int64_t>(b) * p.Hq + h) * p.Lq + row, m, log2f(l),
                                 none);
            tc::fence_before();
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFwdOtherRegs));
        if (warp == 4 && lane == 0 && j0 < j1) {
            bool alive = true;
            int copies = 0;
            mbar_arrive_expect_tx(&bars.q, S::tile);
            load_rows<DP>(Qs, &mq, &bars.q, h, q0, b);
            int issued = 0, k_issued = 0;   // values, keys
            for (int j = j0; j < j1; ++j, ++issued) {
                const int s = issued % NS;
                if (issued >= NS) alive = wait(&bars.k_empty[s], (issued / NS - 1) & 1);
                if (!alive) break;
                mbar_arrive_expect_tx(&bars.k_full[s], S::block);
                ++k_issued;
                if (copies++ == bnd.skip) break;
                load_rows<DP, kKeys>(K_at(s), &mk, &bars.k_full[s], hk, j * kKeys, b);
                if (issued >= NS) alive = wait(&bars.v_empty[s], (issued / NS - 1) & 1);
                if (!alive) break;
                mbar_arrive_expect_tx(&bars.v_full[s], S::block);
                load_rows<DP, kKeys>(V_at(s), &mv, &bars.v_full[s], hk, j * kKeys, b);
            }
            // every copy has landed before the block may end
            mbar_wait32(smem_u32(&bars.q), 0, bnd.timeouts);
            for (int i = max(0, k_issued - NS); i < k_issued; ++i)
                if (bnd.skip < 0 || i != bnd.skip)
                    mbar_wait32(smem_u32(&bars.k_full[i % NS]), (i / NS) & 1, bnd.timeouts);
            for (int i = max(0, issued - NS); i < issued; ++i)
                mbar_wait32(smem_u32(&bars.v_full[i % NS]), (i / NS) & 1, bnd.timeouts);
        } else if (warp == 5 && j0 < j1) {
            const uint32_t iqk = tc::product(kBf16, 128, kKeys, false, false);
            const uint32_t ipv = tc::product(kBf16, 128, cols, false, true);
            const uint32_t q = smem_u32(Qs);
            const bool lead = tc::elect();
            bool fine = wait(&bars.q, 0);
            int st = 0, phase = 0, last = 0, last_phase = 0;   // ring stage and phase of block j + 1; of j
            for (int j = j0 - 1; j < j1; ++j) {
                const int n = j + 1 - j0, c = j - j0;
                if (j + 1 < j1) {
                    // (a block that needs no guard: its keys are enough)
                    fine &= wait(guarded(j + 1) ? &bars.ok[st] : &bars.k_full[st], phase);
                    // S(n) in the place of S and P of the block before last, once PV has read that
                    if (n > 1) fine &= wait(&bars.pv, n & 1);
                    tc::fence_after();
                    if (lead) {
                        scores_mma<DP, kKeys>(tmem + (n & 1) * kKeys, q, smem_u32(K_at(st)), iqk, steps);
                        tc::commit(smem_u32(&bars.s_full[n & 1]));
                        tc::commit(smem_u32(&bars.k_empty[st]));
                    }
                }
                if (j >= j0) {
                    fine &= wait(&bars.ok[last], last_phase);
                    fine &= wait(&bars.p_full[c & 1], (c >> 1) & 1);
                    tc::fence_after();
                    if (lead) {
                        const uint32_t w = tmem + (c & 1) * kKeys, v = smem_u32(V_at(last));
                        mix_mma<4, 4, 0>(tmem + 128, w, v, S::panel, ipv, c > 0);
                        if (REST) mix_mma<4, 4, 0>(tmem + 128, w + 32, v, S::panel, ipv, true);
                        tc::commit(smem_u32(&bars.pv));
                        tc::commit(smem_u32(&bars.v_empty[last]));
                        if (j + 1 == j1) tc::commit(smem_u32(&bars.o_full));
                    }
                }
                last = st;
                last_phase = phase;
                if (++st == NS) {
                    st = 0;
                    phase ^= 1;
                }
                if (!__all_sync(0xffffffffu, fine)) break;
            }
            if (!__all_sync(0xffffffffu, fine)) {   // the products in flight read this block's memory
                if (lead) tc::commit(smem_u32(&bars.drain));
                mbar_wait32(smem_u32(&bars.drain), 0, bnd.timeouts);
            }
        } else if (warp == 7 && j0 < j1) {
            // Every block is passed on: PV waits for that, so no value block is replaced
            // before it was looked at, and no phase of a barrier is taken for another.
            int i = 0;
            for (int j = j0; j < j1; ++j, ++i) {
                const int s = i % NS;
                const uint32_t parity = (i / NS) & 1;
                if (!wait(&bars.v_full[s], parity)) break;
                if (guarded(j) && !wait(&bars.k_full[s], parity)) break;
                if (guarded(j)) {
                    const uint32_t bad = scrub_rows<T, DP, kKeys>(V_at(s), lane, 32);
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        if (bad >> r & 1) poison_row<DP, kKeys>(K_at(s), lane + 32 * r);
                    fence_async_shared();
                }
                mbar_arrive(&bars.ok[s]);
            }
        }
        __syncwarp();
    }
    __syncthreads();
    if (warp == 5) {
        tc::fence_after();
        tc::tmem_free(tmem, 256);
    }
}

template <typename T, int DP, bool CAP, bool BIAS, bool REST>
nsc_status tc_fwd_launch(const Params& p, cudaStream_t st) {
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    auto kern = tc_fwd_kernel<T, DP, CAP, BIAS, REST>;
    const int smem = FwdShape<DP>::smem + 1024 + (BIAS ? 4 * (2 * p.reach + 2 * kBiasPad + 1) : 0);
    nsc_status ready = raise_shared("token_attention", reinterpret_cast<const void*>(kern), smem, kFwdThreads,
                                    128 * kFwdMathRegs + 128 * kFwdOtherRegs);
    if (ready != NSC_OK) return ready;
    CUtensorMap mq, mk, mv;
    const char* err = nullptr;
    if (!encode_heads(&mq, p.q, p.qs, p.B, p.Lq, p.Hq, p.D, kBf16, &err) ||
        !encode_heads(&mk, p.k, p.ks, p.B, p.Lk, p.Hkv, p.D, kBf16, &err, kKeys) ||
        !encode_heads(&mv, p.v, p.vs, p.B, p.Lk, p.Hkv, p.D, kBf16, &err, kKeys))
        return fail(NSC_ERR_LAUNCH_FAILED, "token_attention: %s", err);
    Bounded bnd{wait_timeout_counter(), -1, 0};
    if (!bnd.timeouts)
        return fail(NSC_ERR_LAUNCH_FAILED, "token_attention: no wait counter");
    wait_fault_settings(&bnd.skip, &bnd.budget);
    const int64_t blocks = static_cast<int64_t>((p.Lq + kRows - 1) / kRows) * p.B * p.Hq;
    kern<<<static_cast<unsigned>(blocks), kFwdThreads, smem, st>>>(mq, mk, mv, p, bnd);
    return check_launch("token_attention");
}

}  // namespace

template <typename T, int DP, bool REST>
nsc_status tc_fwd_scores(const Params& p, cudaStream_t st) {
    if (p.cap > 0)
        return p.table ? tc_fwd_launch<T, DP, true, true, REST>(p, st)
                       : tc_fwd_launch<T, DP, true, false, REST>(p, st);
    return p.table ? tc_fwd_launch<T, DP, false, true, REST>(p, st)
                   : tc_fwd_launch<T, DP, false, false, REST>(p, st);
}

template <typename T, int DP>
nsc_status tc_fwd_run(const Params& p, cudaStream_t st) {
    return p.residue ? tc_fwd_scores<T, DP, true>(p, st) : tc_fwd_scores<T, DP, false>(p, st);
}

}  // namespace tok
}  // namespace nsc
