// token_attention_short.cu -- forward of token attention, fp16 / bf16, for few
// tokens (windows, small grids): a block of 4 warps has 64 queries of a head, a warp 16
// of them, and passes the keys 64 at a time.
//
// Bound by latency: such a call is many small heads, each a chain of loads, two small
// products and a softmax.  A 128-row tcgen05 tile would be half empty, and has some 5 us
// of set-up a block with two blocks an SM; here a block takes 3 us or so and three to
// seven share an SM.  256 windows of 64 tokens, 8 heads of 32, with a bias table: 17 us
// (33 MB, 1.9 TB/s) against 38 us; heads of 64: 25 against 40.
// Products are those of a warp (m16n8k16); a row's statistics lie in the four lanes
// that hold its scores.
#include <climits>

#include "token_warp_mma.cuh"

namespace nsc {
namespace tok {
namespace {

constexpr int kShortThreads = 128;
constexpr int kKeys = 64;

template <typename T, int DP, bool CAP, bool BIAS, bool REST>
__global__ __launch_bounds__(kShortThreads, DP == 32 ? 7 : DP == 64 ? 5 : 3) void short_fwd_kernel(const Params p) {
    constexpr int LD = 2 * DP + 16, KS = DP / 16, CH = DP / 8;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int box[4];
    __shared__ unsigned long long odd_keys;
    unsigned char* Ks = smem;
    unsigned char* Vs = smem + kKeys * LD;
    float* E = reinterpret_cast<float*>(smem + 2 * kKeys * LD);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, sub = lane & 3;
    const int nt = (p.Lq + 63) / 64;
    const int64_t id = blockIdx.x;
    const int t = static_cast<int>(id % nt);
    const int bh = static_cast<int>(id / nt), b = bh / p.Hq, h = bh % p.Hq, hk = h / p.G;
    const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[2];
    const T* kb = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
    const T* vb = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
    const int off = p.Lk - p.Lq;

    if (threadIdx.x < 4) box[threadIdx.x] = threadIdx.x == 0 || threadIdx.x == 3 ? INT_MAX : 0;
    __syncthreads();
    int lo[2], hi[2], row[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        row[x] = t * 64 + warp * 16 + quad + 8 * x;
        lo[x] = hi[x] = 0;
        if (row[x] < p.Lq) key_span(p, b, row[x], p.Lk, lo[x], hi[x]);
    }
    {
        const bool a0 = hi[0] > lo[0], a1 = hi[1] > lo[1];
        const int v0 = __reduce_min_sync(~0u, min(a0 ? lo[0] : INT_MAX, a1 ? lo[1] : INT_MAX));
        const int v1 = __reduce_max_sync(~0u, max(a0 ? hi[0] : 0, a1 ? hi[1] : 0));
        const int v2 = __reduce_max_sync(~0u, max(a0 ? lo[0] : 0, a1 ? lo[1] : 0));
        const int v3 = __reduce_min_sync(~0u, min(a0 ? hi[0] : INT_MAX, a1 ? hi[1] : INT_MAX));
        if (lane == 0) {
            atomicMin(&box[0], v0);
            atomicMax(&box[1], v1);
            atomicMax(&box[2], v2);
            atomicMin(&box[3], v3);
        }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)   // (a row past the end is not written: no masks for its sake)
        if (row[x] >= p.Lq) hi[x] = INT_MAX;
    uint32_t qa[KS][4];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int d = 16 * s + 8 * y + 2 * sub;
                qa[s][x + 2 * y] =
                    row[x] < p.Lq && d < p.D
                        ? __ldg(reinterpret_cast<const uint32_t*>(q + row[x] * p.qs[1] + d))
                        : 0u;
            }
    if (BIAS)
        for (int i = threadIdx.x; i <= 2 * p.reach; i += kShortThreads)
            E[i] = bias2_at<float>(p, __ldg(p.lut + i), h);
    __syncthreads();
    const int first = box[0], last = box[1], all_lo = box[2], all_hi = box[3];

    const float unit = static_cast<float>((CAP ? p.cap : p.scale) * kLog2e);
    const float y1 = CAP ? static_cast<float>(p.scale / p.cap) : 0.f;
    float o[2 * KS][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2 * KS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    const uint32_t ka = smem_u32(Ks) + (((lane >> 4) & 1) * 8 + (lane & 7)) * LD + ((lane >> 3) & 1) * 16;
    const uint32_t va = smem_u32(Vs) + (((lane >> 3) & 1) * 8 + (lane & 7)) * LD + (lane >> 4) * 16;

    for (int k0 = first / kKeys * kKeys; k0 < last; k0 += kKeys) {
        __syncthreads();   // (the last block's tiles and its odd_keys are used up)
        if (threadIdx.x == 0) odd_keys = 0;
        for (int u = threadIdx.x; u < kKeys * CH; u += kShortThreads) {
            const int r = u / CH, c = u % CH;
            const bool in = k0 + r < p.Lk && 8 * c < p.D;
            const int64_t key = in ? k0 + r : 0;
            const int d = in ? 8 * c : 0;
            copy16(smem_u32(Ks) + r * LD + 16 * c, kb + key * p.ks[1] + d, in);
            copy16(smem_u32(Vs) + r * LD + 16 * c, vb + key * p.vs[1] + d, in);
        }
        copies_commit();
        copies_wait<0>();
        __syncthreads();
        // where some row does not see the whole block: a value row that is not finite
        // becomes zero, and its key's scores NaN where it is seen
        const bool part = k0 < all_lo || min(k0 + kKeys, p.Lk) > all_hi;
        if (part) {
            bool bad = false;
            const int r = threadIdx.x >> 1;
            uint4* v = reinterpret_cast<uint4*>(Vs + r * LD + (threadIdx.x & 1) * DP);
            const uint32_t ex = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
                const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) bad |= (w[e] & ex) == ex || (w[e] >> 16 & ex) == ex;
            }
            if (__syncthreads_or(bad)) {
                if (bad) atomicOr(&odd_keys, 1ull << r);
                __syncthreads();
                if (odd_keys >> r & 1)
                    for (int c = 0; c < DP / 16; ++c) v[c] = make_uint4(0, 0, 0, 0);
                __syncthreads();
            }
        }
        const unsigned long long odd = odd_keys;
        // Whether some row of this warp does not see all 64 keys.  (`part` does not tell: it
        // is of the rows that see anything, and of the keys there are.)
        const bool hide = __any_sync(~0u, max(lo[0], lo[1]) > k0 || min(hi[0], hi[1]) < k0 + kKeys);
        float s[8][4];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t f[4];
                ldm4(ka + i * 16 * LD + 32 * c, f);
                mma16816<T>(s[2 * i], qa[c], f[0], f[1]);
                mma16816<T>(s[2 * i + 1], qa[c], f[2], f[3]);
            }
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int x = e >> 1, c = 8 * i + 2 * sub + (e & 1), key = k0 + c;
                float v = (CAP ? tanh_exact(s[i][e] * y1) : s[i][e]) * unit;
                if (BIAS) v += E[min(max(key - (row[x] + off), -p.reach), p.reach) + p.reach];
                if (hide) {
                    if (odd >> c & 1) v = NAN;
                    if (key < lo[x] || key >= hi[x]) v = -INFINITY;
                }
                s[i][e] = v;
                top[x] = fmaxf(top[x], v);
            }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            top[x] = fmaxf(top[x], __shfl_xor_sync(~0u, top[x], 1));
            top[x] = fmaxf(top[x], __shfl_xor_sync(~0u, top[x], 2));
            const float mn = fmaxf(m[x], top[x]);
            const float keep = m[x] == -INFINITY ? 0.f : tc::ex2(m[x] - mn);
            m[x] = mn;
            l[x] *= keep;
#pragma unroll
            for (int c = 0; c < 2 * KS; ++c) {
                o[c][2 * x] *= keep;
                o[c][2 * x + 1] *= keep;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // 16 keys
            uint32_t pa[4], rest[4];
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float ref = m[x] == -INFINITY ? 0.f : m[x];
                    const float e0 = tc::ex2(s[2 * i + y][2 * x] - ref);
                    const float e1 = tc::ex2(s[2 * i + y][2 * x + 1] - ref);
                    l[x] += e0 + e1;
                    pa[2 * y + x] = tc::pack2<T>(e0, e1);
                    if (REST) rest[2 * y + x] = tc::rest2<T>(make_float2(e0, e1), pa[2 * y + x]);
                }
#pragma unroll
            for (int c = 0; c < KS; ++c) {
                uint32_t f[4];
                ldm4t(va + i * 16 * LD + 32 * c, f);
                mma16816<T>(o[2 * c], pa, f[0], f[1]);
                mma16816<T>(o[2 * c + 1], pa, f[2], f[3]);
                if (REST) {   // see the tensor-core forward
                    mma16816<T>(o[2 * c], rest, f[0], f[1]);
                    mma16816<T>(o[2 * c + 1], rest, f[2], f[3]);
                }
            }
        }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        l[x] += __shfl_xor_sync(~0u, l[x], 1);
        l[x] += __shfl_xor_sync(~0u, l[x], 2);
        if (row[x] >= p.Lq) continue;
        const bool none = l[x] == 0.f;
        const float inv = none ? 0.f : 1.f / l[x];
        const int64_t at = ((static_cast<int64_t>(b) * p.Lq + row[x]) * p.Hq + h) * p.D;
#pragma unroll
        for (int c = 0; c < 2 * KS; ++c) {
            const int d = 8 * c + 2 * sub;
            if (d >= p.D) break;
            const float u = none ? 0.f : o[c][2 * x] * inv, v = none ? 0.f : o[c][2 * x + 1] * inv;
            const uint32_t w = tc::pack2<T>(u, v);
            *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + at + d) = w;
            if (REST) {
                const T* back = reinterpret_cast<const T*>(&w);
                *reinterpret_cast<uint32_t*>(static_cast<T*>(p.residue) + at + d) =
                    tc::pack2<T>(u - to_acc(back[0]), v - to_acc(back[1]));
            }
        }
        if (sub == 0)
            row_stats<float>(p, static_cast<int64_t>(bh) * p.Lq + row[x], m[x], log2f(l[x]), none);
    }
}

template <typename T, int DP, bool CAP, bool BIAS, bool REST>
nsc_status launch(const Params& p, cudaStream_t st) {
    auto kern = short_fwd_kernel<T, DP, CAP, BIAS, REST>;
    // at most 35 KB of tiles and 8 KB of bias: no opt-in is needed
    const int smem = 2 * kKeys * (2 * DP + 16) + (BIAS ? 4 * (2 * p.reach + 1) : 0);
    const int64_t blocks = static_cast<int64_t>(p.B) * p.Hq * ((p.Lq + 63) / 64);
    kern<<<static_cast<unsigned>(blocks), kShortThreads, smem, st>>>(p);
    return check_launch("token_attention");
}
template <typename T, int DP, bool REST>
nsc_status run(const Params& p, cudaStream_t st) {
    if (p.cap > 0)
        return p.table ? launch<T, DP, true, true, REST>(p, st)
                       : launch<T, DP, true, false, REST>(p, st);
    return p.table ? launch<T, DP, false, true, REST>(p, st)
                   : launch<T, DP, false, false, REST>(p, st);
}
template <typename T, bool REST>
nsc_status run(const Params& p, cudaStream_t st) {
    return p.D <= 32   ? run<T, 32, REST>(p, st)
           : p.D <= 64 ? run<T, 64, REST>(p, st)
                       : run<T, 128, REST>(p, st);
}

}  // namespace

// At most 64 tokens, or 128 with heads of at most 32, in a layout that tc_fits.  Measured
// against the 128-row tiles, 8 heads: 64 tokens 17 / 38 us (heads of 32), 25 / 40 (64),
// 52 / 51 (128; 33 tokens 40 / 46); 170 x 100 tokens 34 / 35, 48 / 37 and 91 / 49.
bool short_fits(const Params& p, int dtype) {
    const int most = p.D <= 32 ? 128 : 64;
    return tc_fits(p, dtype) && p.Lk <= most && p.Lq <= most;
}

nsc_status short_fwd(const Params& p, int dtype, cudaStream_t st) {
    if (p.residue)
        return dtype == NSC_BF16 ? run<__nv_bfloat16, true>(p, st) : run<__half, true>(p, st);
    return dtype == NSC_BF16 ? run<__nv_bfloat16, false>(p, st) : run<__half, false>(p, st);
}

}  // namespace tok
}  // namespace nsc
