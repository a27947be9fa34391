// token_decode.cu -- token attention of the newest tokens over ragged caches.
//
// Bound by memory: every key and value of a cache is read once for all G T rows
// (query heads that share the key head, times new tokens) of its head.  The long
// axis is cut into chunks, a block each, so that a few long sequences fill the
// GPU as many short ones do; a block leaves an unnormalised output row with its
// reference m and sum l, and a second kernel joins a row's chunks:
//     out = sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c
// (a call whose caches are one chunk long writes its output at once).
//
// decode_mma_kernel (fp16 / bf16): 4 warps, each with its own ring of 16 keys and
// values filled by asynchronous 16-byte copies, so that no barrier stands between a
// warp and its memory; scores and outputs of 16 or 32 rows by 16-bit tensor-core
// products of a warp, statistics in fp32.  A tile of tcgen05 would be 128 rows for
// the few there are.  Two blocks an SM (three at D <= 64): one joins its warps'
// outputs while the other reads.
// 32 ragged caches to 8192 keys, 32 / 8 heads of 128, capped, bf16: 82 us for 500 MB
// (6.0 TB/s), the join 7; two caches of 65530 keys, 16 / 2 heads of 128, 4 new tokens,
// fp16: 36 us (3.8 TB/s: a block's start and end beside its 450 keys), the join 7.
// decode_f32_kernel: fp32 on the FMA pipes, 4 or 8 rows a block, in registers.
// decode_any_kernel: any type, width and alignment, 8 rows a block, tile by tile through
// shared memory.
#include <algorithm>
#include <type_traits>

#include "token_warp_mma.cuh"

namespace nsc {
namespace tok {
namespace {

constexpr int kWarps = 4;            // of a tensor-core block
constexpr int kMmaThreads = 32 * kWarps;
constexpr int kF32Threads = 128;
constexpr int kThreads = 256;        // of the others
constexpr float kLazyMove = 8.f;

struct Split {
    int chunk, n_chunk;   // keys of a chunk, chunks of a cache
    int groups, stages;   // row groups of a head, ring depth
    void* part;           // (rows, n_chunk, wide) outputs, then (rows, n_chunk, 2) m, l
};
__host__ __device__ __forceinline__ int part_wide(int D) { return (D + 3) / 4 * 4; }
template <typename A>
__device__ __forceinline__ A* part_ml(const Params& p, const Split& sp) {
    return static_cast<A*>(sp.part) +
           static_cast<int64_t>(p.B) * p.Hq * p.Lq * sp.n_chunk * part_wide(p.D);
}
template <typename A>
__device__ __forceinline__ void put_part(const Params& p, const Split& sp, int64_t row, int chunk,
                                         int d, A v, A m, A l) {
    const int64_t at = row * sp.n_chunk + chunk;
    static_cast<A*>(sp.part)[at * part_wide(p.D) + d] = v;
    if (d == 0) {
        part_ml<A>(p, sp)[2 * at] = m;
        part_ml<A>(p, sp)[2 * at + 1] = l;
    }
}

// Row r of a head's G T rows: query head hk G + r / T, new token r % T.
__device__ __forceinline__ void row_of(const Params& p, int hk, int r, int& h, int& t) {
    h = hk * p.G + r / p.Lq;
    t = r - r / p.Lq * p.Lq;
}

// The last key that new token t sees, of n.
__device__ __forceinline__ int last_seen(const Params& p, int n, int t) {
    return p.causal ? n - p.Lq + t : n - 1;
}

template <typename T, int DP, int MT, int NS, bool CAP, bool BIAS>
__global__ __launch_bounds__(kMmaThreads, DP == 64 ? 3 : 2) void decode_mma_kernel(const Params p, const Split sp) {
    constexpr int LD = 2 * DP + 16;        // bytes of a row: rows 16 bytes apart in the banks
    constexpr int TILE = 16 * LD;          // 16 keys, or values
    constexpr int KS = DP / 16;
    constexpr int R = 16 * MT;             // rows of the block
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float ms[kWarps][R], ls[kWarps][R];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, sub = lane & 3;
    int id = blockIdx.x;
    const int chunk = id % sp.n_chunk;
    id /= sp.n_chunk;
    const int group = id % sp.groups;
    id /= sp.groups;
    const int hk = id % p.Hkv, b = id / p.Hkv;
    const int n = keys_of(p, b), c0 = chunk * sp.chunk, c1 = min(n, c0 + sp.chunk);
    if (c0 >= n && chunk > 0) return;
    const int rows = p.G * p.Lq, r0 = group * R;

    unsigned char* Qs = smem + kWarps * NS * 2 * TILE;   // [R][LD], where MT > 1
    float* table = reinterpret_cast<float*>(Qs + (MT > 1 ? R * LD : 0));
    unsigned char* bucket = reinterpret_cast<unsigned char*>(table);
    const int first_head = r0 / p.Lq, heads = min(p.G - 1, (r0 + R - 1) / p.Lq) - first_head + 1;
    // keys from `near` on are within reach of some new token
    const int near = n - p.Lq - p.reach;
    if (BIAS) {
        bucket += sizeof(float) * heads * p.nb;
        if (c1 > near) {
            for (int i = threadIdx.x; i < heads * p.nb; i += kMmaThreads)
                table[i] = bias2_at<float>(p, i % p.nb, hk * p.G + first_head + i / p.nb);
            for (int i = threadIdx.x; i <= p.reach; i += kMmaThreads)
                bucket[i] = static_cast<unsigned char>(
                    min(max(__ldg(p.lut + p.reach - i), 0), p.nb - 1));
        }
        __syncthreads();
    }

    const T* kb = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
    const T* vb = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
    const uint32_t ring = smem_u32(smem) + warp * NS * 2 * TILE;
    const int k_first = c0 + 16 * warp;
    const int steps = c1 > k_first ? (c1 - k_first + 16 * kWarps - 1) / (16 * kWarps) : 0;
    // a lane copies one 16-byte column of every (32 / columns)th row; columns past D are zero
    constexpr int CH = DP / 8, RS = 32 / CH;   // columns of a row, rows a pass
    const int cr = lane / CH, cc = lane % CH;
    const bool c_in = 8 * cc < p.D;
    const int64_t k_pass = RS * p.ks[1], v_pass = RS * p.vs[1];
    const T* k_src = kb + static_cast<int64_t>(min(k_first + cr, n - 1)) * p.ks[1] + (c_in ? 8 * cc : 0);
    const T* v_src = vb + static_cast<int64_t>(min(k_first + cr, n - 1)) * p.vs[1] + (c_in ? 8 * cc : 0);
    const int64_t k_step = 16 * kWarps * p.ks[1], v_step = 16 * kWarps * p.vs[1];
    const uint32_t c_dst = ring + cr * LD + 16 * cc;
    int put = 0, put_stage = 0;
    auto issue = [&]() {
        if (put < steps) {
            const uint32_t dst = c_dst + put_stage * 2 * TILE;
            const int left = c1 - (k_first + 16 * kWarps * put);   // keys of this step
            if (left >= 16) {
                const T *ks = k_src, *vs = v_src;
#pragma unroll
                for (int x = 0; x < 16 / RS; ++x, ks += k_pass, vs += v_pass) {
                    copy16(dst + x * RS * LD, ks, c_in);
                    copy16(dst + TILE + x * RS * LD, vs, c_in);
                }
            } else {
#pragma unroll
                for (int x = 0; x < 16 / RS; ++x) {
                    const bool in = c_in && cr + RS * x < left;
                    copy16(dst + x * RS * LD, in ? k_src + x * k_pass : kb, in);
                    copy16(dst + TILE + x * RS * LD, in ? v_src + x * v_pass : vb, in);
                }
            }
            k_src += k_step;
            v_src += v_step;
        }
        ++put;
        put_stage = put_stage + 1 == NS ? 0 : put_stage + 1;
        copies_commit();
    };
#pragma unroll
    for (int i = 0; i < NS; ++i) issue();

    // the rows' queries as A operands: in registers, or (two tiles) in shared memory
    uint32_t qa[MT > 1 ? 1 : KS][4];
    int pos[2 * MT], head[2 * MT];
    float e_far[2 * MT];
    if (MT > 1) {
#pragma unroll 2
        for (int i = warp; i < R; i += kWarps) {   // a warp a row
            const int r = r0 + i;
            int h = 0, t = 0;
            if (r < rows) row_of(p, hk, r, h, t);
            const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + t * p.qs[1] + h * p.qs[2];
#pragma unroll
            for (int d = 2 * lane; d < DP; d += 64)
                *reinterpret_cast<uint32_t*>(Qs + i * LD + 2 * d) =
                    r < rows && d < p.D ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
        }
        __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < 2 * MT; ++x) {
        const int r = r0 + quad + 8 * x;
        int h = 0, t = 0;
        const bool in = r < rows;
        if (in) row_of(p, hk, r, h, t);
        pos[x] = in ? last_seen(p, n, t) : -1;
        e_far[x] = 0.f;
        head[x] = 0;
        if (BIAS && in) {
            e_far[x] = bias2_at<float>(p, __ldg(p.lut), h);
            head[x] = h - hk * p.G - first_head;
        }
        if (MT == 1) {
            const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + t * p.qs[1] + h * p.qs[2];
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const int d = 16 * s + 8 * y + 2 * sub;
                    qa[MT > 1 ? 0 : s][x + 2 * y] =
                        in && d < p.D ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
                }
        }
    }
    const uint32_t q_at = smem_u32(Qs) + (lane & 15) * LD + (lane >> 4) * 16;
    const float unit = static_cast<float>((CAP ? p.cap : p.scale) * kLog2e);
    const float y1 = CAP ? static_cast<float>(p.scale / p.cap) : 0.f;
    float o[MT][2 * KS][4], m[2 * MT], l[2 * MT];
#pragma unroll
    for (int x = 0; x < 2 * MT; ++x) {
        m[x] = -INFINITY;
        l[x] = 0.f;
    }
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[a][i][e] = 0.f;

    for (int i = 0, stage = 0; i < steps; ++i, stage = stage + 1 == NS ? 0 : stage + 1) {
        copies_wait<NS - 1>();
        __syncwarp();
        const int k0 = k_first + 16 * kWarps * i;
        const uint32_t kt = ring + stage * 2 * TILE, vt = kt + TILE;
        float s[MT][2][4];
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[a][y][e] = 0.f;
        const uint32_t ka = kt + (((lane >> 4) & 1) * 8 + (lane & 7)) * LD + ((lane >> 3) & 1) * 16;
#pragma unroll
        for (int c = 0; c < KS; ++c) {
            uint32_t f[4];
            ldm4(ka + 32 * c, f);
#pragma unroll
            for (int a = 0; a < MT; ++a) {
                uint32_t w[4];
                if (MT > 1) ldm4(q_at + 16 * a * LD + 32 * c, w);
                mma16816<T>(s[a][0], MT > 1 ? w : qa[MT > 1 ? 0 : c], f[0], f[1]);
                mma16816<T>(s[a][1], MT > 1 ? w : qa[MT > 1 ? 0 : c], f[2], f[3]);
            }
        }
        // past the oldest new token's position some row does not see a key: a value
        // there that is not finite becomes zero, and NaN scores where it is seen
        const bool tail = k0 + 16 > n - p.Lq + 1;
        uint32_t odd = 0;
        if (tail && p.Lq > 1) {
            const int r = lane >> 1;
            const uint4* row = reinterpret_cast<const uint4*>(smem + (vt - smem_u32(smem)) + r * LD +
                                                              (lane & 1) * DP);
            bool bad = false;
            for (int c = 0; c < DP / 16; ++c) {
                const uint4 v = row[c];
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t ex = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
                    bad |= (w[e] & ex) == ex || (w[e] >> 16 & ex) == ex;
                }
            }
            const uint32_t who = __ballot_sync(0xffffffffu, bad);
            odd = who | (who >> 1 & 0x55555555u) | (who << 1 & 0xAAAAAAAAu);   // both halves of a row
            if (odd >> lane & 1)
                for (int c = 0; c < DP / 16; ++c) const_cast<uint4*>(row)[c] = make_uint4(0, 0, 0, 0);
            __syncwarp();
        }
        // (the rare parts stand apart: folded into one loop they would be issued,
        // predicated off, for every key)
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s[a][y][e] = (CAP ? tanh_exact(s[a][y][e] * y1) : s[a][y][e]) * unit;
        if (BIAS && k0 + 15 >= near) {
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int x = 2 * a + (e >> 1), key = k0 + 8 * y + 2 * sub + (e & 1);
                        const int d = min(max(pos[x] - key, 0), p.reach);
                        s[a][y][e] += table[head[x] * p.nb + bucket[d]];
                    }
        } else if (BIAS) {
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[a][y][e] += e_far[2 * a + (e >> 1)];
        }
        if (tail) {
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int c = 8 * y + 2 * sub + (e & 1);
                        if (odd >> (2 * c) & 1) s[a][y][e] = NAN;
                        if (k0 + c > pos[2 * a + (e >> 1)]) s[a][y][e] = -INFINITY;
                    }
        }
        float top[2 * MT];
#pragma unroll
        for (int x = 0; x < 2 * MT; ++x)
            top[x] = fmaxf(fmaxf(s[x >> 1][0][2 * (x & 1)], s[x >> 1][0][2 * (x & 1) + 1]),
                           fmaxf(s[x >> 1][1][2 * (x & 1)], s[x >> 1][1][2 * (x & 1) + 1]));
        bool moved = false;
        float keep[2 * MT];
#pragma unroll
        for (int x = 0; x < 2 * MT; ++x) {
            top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
            top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
            keep[x] = 1.f;
            if (top[x] > m[x] + kLazyMove || m[x] == -INFINITY) {
                keep[x] = m[x] == -INFINITY ? 0.f : tc::ex2(m[x] - top[x]);
                m[x] = fmaxf(top[x], m[x]);
                moved = true;
            }
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int x = 0; x < 2 * MT; ++x) l[x] *= keep[x];
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int c = 0; c < 2 * KS; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[a][c][e] *= keep[2 * a + (e >> 1)];
        }
        uint32_t pa[MT][4];
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int x = 2 * a + e;
                    const float ref = m[x] == -INFINITY ? 0.f : m[x];
                    const float e0 = tc::ex2(s[a][y][2 * e] - ref);
                    const float e1 = tc::ex2(s[a][y][2 * e + 1] - ref);
                    l[x] += e0 + e1;
                    pa[a][2 * y + e] = tc::pack2<T>(e0, e1);
                }
        const uint32_t va = vt + (((lane >> 3) & 1) * 8 + (lane & 7)) * LD + (lane >> 4) * 16;
#pragma unroll
        for (int c = 0; c < KS; ++c) {
            uint32_t f[4];
            ldm4t(va + 32 * c, f);
#pragma unroll
            for (int a = 0; a < MT; ++a) {
                mma16816<T>(o[a][2 * c], pa[a], f[0], f[1]);
                mma16816<T>(o[a][2 * c + 1], pa[a], f[2], f[3]);
            }
        }
        __syncwarp();
        issue();
    }
    copies_wait<0>();
#pragma unroll
    for (int x = 0; x < 2 * MT; ++x) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
        if (sub == 0) {
            ms[warp][quad + 8 * x] = m[x];
            ls[warp][quad + 8 * x] = l[x];
        }
    }
    __syncthreads();   // (every warp is done with its ring)
    float* sh = reinterpret_cast<float*>(smem);   // [warps][R][DP + 4]
    constexpr int LO = DP + 4;
#pragma unroll
    for (int x = 0; x < 2 * MT; ++x) {
        float M = -INFINITY;
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ms[w][quad + 8 * x]);
        const float f = m[x] == -INFINITY ? 0.f : tc::ex2(m[x] - M);
#pragma unroll
        for (int c = 0; c < 2 * KS; ++c) {
            float* at = sh + (warp * R + quad + 8 * x) * LO + 8 * c + 2 * sub;
            // (a row without weight may hold NaN products only where l is NaN)
            at[0] = f == 0.f && l[x] == 0.f ? 0.f : o[x >> 1][c][2 * (x & 1)] * f;
            at[1] = f == 0.f && l[x] == 0.f ? 0.f : o[x >> 1][c][2 * (x & 1) + 1] * f;
        }
    }
    __syncthreads();
    // a warp a row, four channels a lane
#pragma unroll 2
    for (int r = warp; r < R; r += kWarps) {
        if (r0 + r >= rows) break;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ms[w][r]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w)   // (a warp without weight: l is zero, or NaN)
            L += ms[w][r] == -INFINITY ? ls[w][r] : ls[w][r] * tc::ex2(ms[w][r] - M);
        int h, t;
        row_of(p, hk, r0 + r, h, t);
        const int64_t row = (static_cast<int64_t>(b) * p.Hq + h) * p.Lq + t;
        const int64_t at = row * sp.n_chunk + chunk;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        if (4 * lane < p.D) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float4 x = *reinterpret_cast<const float4*>(sh + (w * R + r) * LO + 4 * lane);
                v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
            }
            if (sp.n_chunk == 1) {
                T* dst = static_cast<T*>(p.out) +
                         ((static_cast<int64_t>(b) * p.Lq + t) * p.Hq + h) * p.D + 4 * lane;
                // (a row that sees nothing may have products of NaN values with zero)
                *reinterpret_cast<uint2*>(dst) =
                    L == 0.f ? make_uint2(0u, 0u)
                             : make_uint2(tc::pack2<T>(v.x * inv, v.y * inv),
                                          tc::pack2<T>(v.z * inv, v.w * inv));
            } else {
                *reinterpret_cast<float4*>(static_cast<float*>(sp.part) + at * p.D + 4 * lane) = v;
            }
        }
        if (lane == 0) {
            if (sp.n_chunk == 1) {
                row_stats<float>(p, row, M, log2f(L), L == 0.f);
            } else {
                part_ml<float>(p, sp)[2 * at] = M;
                part_ml<float>(p, sp)[2 * at + 1] = L;
            }
        }
    }
}

constexpr int kAnyRows = 8, kAnyKeys = 64;

template <typename T, typename A> struct AnyShape {
    static size_t smem(int D) {
        return sizeof(A) * (static_cast<size_t>(kAnyKeys) * (D + 1) * 2 + kAnyRows * D +
                            2 * kAnyRows * kAnyKeys + kThreads * kAnyRows);
    }
};

__device__ __forceinline__ float exp2_any(float x) { return exp2f(x); }
__device__ __forceinline__ double exp2_any(double x) { return exp2(x); }
__device__ __forceinline__ float log2_any(float x) { return log2f(x); }
__device__ __forceinline__ double log2_any(double x) { return log2(x); }
__device__ __forceinline__ float tanh_any(float x) { return tanhf(x); }
__device__ __forceinline__ double tanh_any(double x) { return tanh(x); }
template <typename T> __device__ __forceinline__ T as_type(float v) { return from_float<T>(v); }
template <typename T> __device__ __forceinline__ T as_type(double v) { return v; }

template <typename T, typename A>
__global__ __launch_bounds__(kThreads) void decode_any_kernel(const Params p, const Split sp) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ A ref[kAnyRows], keep[kAnyRows], sum[kAnyRows];
    const int D = p.D, LD = D + 1;
    A* Ks = reinterpret_cast<A*>(smem);
    A* Vs = Ks + kAnyKeys * LD;
    A* Qs = Vs + kAnyKeys * LD;
    A* Ss = Qs + kAnyRows * D;                 // [rows][keys]
    A* Ps = Ss + kAnyRows * kAnyKeys;          // [keys][rows]
    A* Os = Ps + kAnyRows * kAnyKeys;          // [threads][rows], at the end
    int id = blockIdx.x;
    const int chunk = id % sp.n_chunk;
    id /= sp.n_chunk;
    const int group = id % sp.groups;
    id /= sp.groups;
    const int hk = id % p.Hkv, b = id / p.Hkv;
    const int n = keys_of(p, b), c0 = chunk * sp.chunk, c1 = min(n, c0 + sp.chunk);
    if (c0 >= n && chunk > 0) return;
    const int rows = p.G * p.Lq, r0 = group * kAnyRows, nr = min(kAnyRows, rows - r0);
    const T* kb = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
    const T* vb = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
    for (int i = threadIdx.x; i < kAnyRows * D; i += kThreads) {
        const int r = i / D, d = i - r * D;
        A v = 0;
        if (r < nr) {
            int h, t;
            row_of(p, hk, r0 + r, h, t);
            v = to_acc(static_cast<const T*>(p.q)[b * p.qs[0] + t * p.qs[1] + h * p.qs[2] + d]);
        }
        Qs[i] = v;
    }
    if (threadIdx.x < kAnyRows) {
        ref[threadIdx.x] = -INFINITY;
        sum[threadIdx.x] = 0;
    }
    // sums of a thread: channel d of kAnyRows rows over a share of the keys
    const int wide = (D + 31) / 32 * 32, shares = kThreads / wide;
    const int d = threadIdx.x % wide, share = threadIdx.x / wide;
    A acc[kAnyRows];
#pragma unroll
    for (int r = 0; r < kAnyRows; ++r) acc[r] = 0;
    const A unit = (p.cap > 0 ? p.cap : p.scale) * kLog2e, y1 = p.cap > 0 ? p.scale / p.cap : 0;
    for (int k0 = c0; k0 < c1; k0 += kAnyKeys) {
        __syncthreads();
        bool odd = false;
        for (int i = threadIdx.x; i < kAnyKeys * D; i += kThreads) {
            const int r = i / D, e = i - r * D;
            A x = 0, y = 0;
            if (k0 + r < c1) {
                x = to_acc(kb[static_cast<int64_t>(k0 + r) * p.ks[1] + e]);
                y = to_acc(vb[static_cast<int64_t>(k0 + r) * p.vs[1] + e]);
            }
            odd |= !(y - y == A(0));
            Ks[r * LD + e] = x;
            Vs[r * LD + e] = y;
        }
        const bool strict = __syncthreads_or(odd);
        {   // scores: thread (key, two rows)
            const int key = threadIdx.x % kAnyKeys, r = threadIdx.x / kAnyKeys * 2;
            A x0 = 0, x1 = 0;
            for (int e = 0; e < D; ++e) {
                const A kv = Ks[key * LD + e];
                x0 += kv * Qs[r * D + e];
                x1 += kv * Qs[(r + 1) * D + e];
            }
            const A x[2] = {x0, x1};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                A v = -INFINITY;
                if (r + i < nr) {
                    int h, t;
                    row_of(p, hk, r0 + r + i, h, t);
                    const int rel = k0 + key - last_seen(p, n, t);
                    if (rel <= 0 && k0 + key < c1) {
                        v = (p.cap > 0 ? tanh_any(x[i] * y1) : x[i]) * unit;
                        if (p.table)
                            v += bias2_at<A>(p, __ldg(p.lut + max(rel, -p.reach) + p.reach), h);
                    }
                }
                Ss[(r + i) * kAnyKeys + key] = v;
            }
        }
        __syncthreads();
        {   // a warp a row
            const int r = threadIdx.x >> 5, lane = threadIdx.x & 31;
            const A a = Ss[r * kAnyKeys + lane], c = Ss[r * kAnyKeys + 32 + lane];
            A top = a > c ? a : c;
#pragma unroll
            for (int i = 16; i; i >>= 1) {
                const A other = __shfl_xor_sync(0xffffffffu, top, i);
                top = other > top ? other : top;
            }
            const A old = ref[r], mn = top > old ? top : old;
            const A base = mn == A(-INFINITY) ? A(0) : mn;
            const A ea = exp2_any(a - base), ec = exp2_any(c - base);
            Ps[lane * kAnyRows + r] = ea;
            Ps[(32 + lane) * kAnyRows + r] = ec;
            A s = ea + ec;
#pragma unroll
            for (int i = 16; i; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
            __syncwarp();
            if (lane == 0) {
                const A f = exp2_any(old - base);
                keep[r] = f;
                ref[r] = mn;
                sum[r] = sum[r] * f + s;
            }
        }
        __syncthreads();
        if (d < D && share < shares) {
#pragma unroll
            for (int r = 0; r < kAnyRows; ++r) acc[r] *= keep[r];
            for (int k = share; k < kAnyKeys; k += shares) {
                const A v = Vs[k * LD + d];
#pragma unroll
                for (int r = 0; r < kAnyRows; ++r) {
                    const A w = Ps[k * kAnyRows + r];
                    if (!strict || w != A(0)) acc[r] += w * v;
                }
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kAnyRows; ++r) Os[threadIdx.x * kAnyRows + r] = acc[r];
    __syncthreads();
    for (int i = threadIdx.x; i < nr * D; i += kThreads) {
        const int r = i / D, e = i - r * D;
        A v = 0;
        for (int s = 0; s < shares; ++s) v += Os[(s * wide + e) * kAnyRows + r];
        const A L = sum[r];
        int h, t;
        row_of(p, hk, r0 + r, h, t);
        const int64_t row = (static_cast<int64_t>(b) * p.Hq + h) * p.Lq + t;
        if (sp.n_chunk == 1) {
            static_cast<T*>(p.out)[((static_cast<int64_t>(b) * p.Lq + t) * p.Hq + h) * D + e] =
                as_type<T>(L == A(0) ? A(0) : v / L);
            if (e == 0) row_stats<A>(p, row, ref[r], log2_any(L), L == A(0));
        } else {
            put_part<A>(p, sp, row, chunk, e, v, ref[r], L);
        }
    }
}

// fp32 rows of 16-byte units, D <= 128: eight lanes a key, D / 8 of its channels a lane, so
// that a warp reads four keys in whole lines; each such group of lanes is a softmax of its
// own (reference, sum and outputs in registers) until the end, so that a key costs three
// exchanges a row and no barrier.  Values are asked for before the scores of their keys,
// keys a step ahead.  RB rows a block.  Bound by memory with few rows: 8 caches of 8192 keys,
// 16 / 4 heads of 128: 66 us for 268 MB (4.0 TB/s; decode_any_kernel 403 us); 32 / 4
// heads 113 us, bound by the FMA pipe.
template <int DP, int RB>
__global__ __launch_bounds__(kF32Threads) void decode_f32_kernel(const Params p, const Split sp) {
    constexpr int C = DP / 32, W = kF32Threads / 32;
    __shared__ __align__(16) float qs[RB][DP];
    __shared__ __align__(16) float os[W][RB][DP];
    __shared__ float ms[W][RB], ls[W][RB];
    __shared__ int row_pos[RB], row_head[RB];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & 7, slot = lane >> 3;
    int id = blockIdx.x;
    const int chunk = id % sp.n_chunk;
    id /= sp.n_chunk;
    const int group = id % sp.groups;
    id /= sp.groups;
    const int hk = id % p.Hkv, b = id / p.Hkv;
    const int n = keys_of(p, b), c0 = chunk * sp.chunk, c1 = min(n, c0 + sp.chunk);
    if (c0 >= n && chunk > 0) return;
    const int rows = p.G * p.Lq, r0 = group * RB, nr = min(RB, rows - r0);
    for (int i = threadIdx.x; i < RB * DP; i += kF32Threads) {
        const int r = i / DP, d = i % DP;
        int h = 0, t = 0;
        if (r < nr) row_of(p, hk, r0 + r, h, t);
        qs[r][d] = r < nr && d < p.D ? static_cast<const float*>(p.q)[b * p.qs[0] + t * p.qs[1] +
                                                                      h * p.qs[2] + d]
                                     : 0.f;
        if (d == 0) {
            row_pos[r] = last_seen(p, n, t);
            row_head[r] = h;
        }
    }
    __syncthreads();
    const float* kb = static_cast<const float*>(p.k) + b * p.ks[0] + hk * p.ks[2] + 4 * sub;
    const float* vb = static_cast<const float*>(p.v) + b * p.vs[0] + hk * p.vs[2] + 4 * sub;
    auto fetch = [&](const float* base, int64_t stride, int key, float4 (&x)[C]) {
#pragma unroll
        for (int j = 0; j < C; ++j)
            x[j] = key < c1 && 4 * sub + 32 * j < p.D
                       ? __ldg(reinterpret_cast<const float4*>(base + key * stride + 32 * j))
                       : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    const float unit = static_cast<float>((p.cap > 0 ? p.cap : p.scale) * kLog2e);
    const float y1 = p.cap > 0 ? static_cast<float>(p.scale / p.cap) : 0.f;
    float acc[RB][4 * C], m[RB], l[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int j = 0; j < 4 * C; ++j) acc[r][j] = 0.f;
    }
    const int first = c0 + 4 * warp, steps = c1 > first ? (c1 - first + 4 * W - 1) / (4 * W) : 0;
    float4 k[C], v[C];
    fetch(kb, p.ks[1], first + slot, k);
    for (int i = 0; i < steps; ++i) {
        const int key = first + 4 * W * i + slot;
        fetch(vb, p.vs[1], key, v);
        float x[RB];
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            float a = 0.f, c = 0.f;
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const float4 q = *reinterpret_cast<const float4*>(&qs[r][4 * sub + 32 * j]);
                a = fmaf(k[j].x, q.x, a);
                c = fmaf(k[j].y, q.y, c);
                a = fmaf(k[j].z, q.z, a);
                c = fmaf(k[j].w, q.w, c);
            }
            x[r] = a + c;
        }
        fetch(kb, p.ks[1], key + 4 * W, k);
#pragma unroll
        for (int e = 1; e < 8; e <<= 1)
#pragma unroll
            for (int r = 0; r < RB; ++r) x[r] += __shfl_xor_sync(0xffffffffu, x[r], e);
        // past the oldest new token's position some row does not see a key
        const bool tail = __any_sync(0xffffffffu, key > n - p.Lq || key >= c1);
        bool moved = false;
        float keep[RB];
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            x[r] = (p.cap > 0 ? tanhf(x[r] * y1) : x[r]) * unit;
            if (p.table) {
                const int rel = min(max(key - row_pos[r], -p.reach), 0);
                x[r] += bias2_at<float>(p, __ldg(p.lut + rel + p.reach), row_head[r]);
            }
            if (tail && (key > row_pos[r] || key >= c1)) x[r] = -INFINITY;
            keep[r] = 1.f;
            if (x[r] > m[r] + kLazyMove || m[r] == -INFINITY) {
                keep[r] = m[r] == -INFINITY ? 0.f : exp2f(m[r] - x[r]);
                m[r] = fmaxf(m[r], x[r]);
                moved = true;
            }
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int r = 0; r < RB; ++r) {
                l[r] *= keep[r];
#pragma unroll
                for (int j = 0; j < 4 * C; ++j) acc[r][j] *= keep[r];
            }
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            x[r] = exp2f(x[r] - (m[r] == -INFINITY ? 0.f : m[r]));
            l[r] += x[r];
        }
        if (tail) {   // (0 x infinity would reach a row that does not see the key)
#pragma unroll
            for (int r = 0; r < RB; ++r)
                if (key <= row_pos[r] && key < c1)
#pragma unroll
                    for (int j = 0; j < C; ++j) {
                        acc[r][4 * j] = fmaf(x[r], v[j].x, acc[r][4 * j]);
                        acc[r][4 * j + 1] = fmaf(x[r], v[j].y, acc[r][4 * j + 1]);
                        acc[r][4 * j + 2] = fmaf(x[r], v[j].z, acc[r][4 * j + 2]);
                        acc[r][4 * j + 3] = fmaf(x[r], v[j].w, acc[r][4 * j + 3]);
                    }
        } else {
#pragma unroll
            for (int r = 0; r < RB; ++r)
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    acc[r][4 * j] = fmaf(x[r], v[j].x, acc[r][4 * j]);
                    acc[r][4 * j + 1] = fmaf(x[r], v[j].y, acc[r][4 * j + 1]);
                    acc[r][4 * j + 2] = fmaf(x[r], v[j].z, acc[r][4 * j + 2]);
                    acc[r][4 * j + 3] = fmaf(x[r], v[j].w, acc[r][4 * j + 3]);
                }
        }
    }
    // the four softmaxes of the warp, then the warps
#pragma unroll
    for (int r = 0; r < RB; ++r) {
        float M = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 8));
        M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 16));
        const float f = m[r] == -INFINITY ? (l[r] == 0.f ? 0.f : 1.f) : exp2f(m[r] - M);
        l[r] *= f;
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 8);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 16);
#pragma unroll
        for (int j = 0; j < 4 * C; ++j) {
            float o = acc[r][j] * f;
            o += __shfl_xor_sync(0xffffffffu, o, 8);
            o += __shfl_xor_sync(0xffffffffu, o, 16);
            if (slot == 0) os[warp][r][4 * sub + 32 * (j / 4) + j % 4] = o;
        }
        if (lane == 0) {
            ms[warp][r] = M;
            ls[warp][r] = l[r];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nr * p.D; i += kF32Threads) {
        const int r = i / p.D, d = i - r * p.D;
        float M = -INFINITY, L = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) M = fmaxf(M, ms[w][r]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = ms[w][r] == -INFINITY ? (ls[w][r] == 0.f ? 0.f : 1.f) : exp2f(ms[w][r] - M);
            L += ls[w][r] * f;
            o += os[w][r][d] * f;
        }
        int h, t;
        row_of(p, hk, r0 + r, h, t);
        const int64_t row = (static_cast<int64_t>(b) * p.Hq + h) * p.Lq + t;
        if (sp.n_chunk == 1) {
            static_cast<float*>(p.out)[((static_cast<int64_t>(b) * p.Lq + t) * p.Hq + h) * p.D + d] =
                L == 0.f ? 0.f : o / L;
            if (d == 0) row_stats<float>(p, row, M, log2f(L), L == 0.f);
        } else {
            put_part<float>(p, sp, row, chunk, d, o, M, L);
        }
    }
}

// A block a row, its warps side by side over the row's chunks, four channels a lane
// at a time.  Bound by latency: the loads of a warp's chunks are independent.
template <typename T, typename A>
__global__ __launch_bounds__(kThreads) void decode_join_kernel(const Params p, const Split sp) {
    constexpr int W = kThreads / 32;
    struct alignas(16) V4 { A v[4]; };
    __shared__ V4 part_o[W][64];
    __shared__ A part_l[W], top[W];
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int bh = row / p.Lq, t = row - bh * p.Lq, b = bh / p.Hq, h = bh - b * p.Hq;
    const int n = keys_of(p, b), used = max(1, (n + sp.chunk - 1) / sp.chunk);
    const int64_t at = static_cast<int64_t>(row) * sp.n_chunk;
    cudaGridDependencySynchronize();   // the chunks' parts are written
    const A* ml = part_ml<A>(p, sp) + 2 * at;
    const V4* o = reinterpret_cast<const V4*>(static_cast<const A*>(sp.part) + at * part_wide(p.D));
    const int wide = part_wide(p.D) / 4;
    A M = -INFINITY;
    for (int c = threadIdx.x; c < used; c += kThreads) {
        const A m = ml[2 * c];
        M = m > M ? m : M;
    }
#pragma unroll
    for (int i = 16; i; i >>= 1) {
        const A x = __shfl_xor_sync(0xffffffffu, M, i);
        M = x > M ? x : M;
    }
    if (lane == 0) top[warp] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) M = top[w] > M ? top[w] : M;
    A L = 0;
    V4 acc[2] = {};
#pragma unroll 8
    for (int c = warp; c < used; c += W) {
        const A m = ml[2 * c], l = ml[2 * c + 1];
        // (a chunk without weight adds nothing; a NaN sum stays one)
        const A f = l == A(0) ? A(0) : m == A(-INFINITY) ? A(1) : exp2_any(m - M);
        L += l * f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (lane + 32 * i < wide) {
                const V4 x = o[static_cast<int64_t>(c) * wide + lane + 32 * i];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i].v[e] += x.v[e] * f;
            }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) part_o[warp][lane + 32 * i] = acc[i];
    if (lane == 0) part_l[warp] = L;
    __syncthreads();
    L = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) L += part_l[w];
    T* dst = static_cast<T*>(p.out) + ((static_cast<int64_t>(b) * p.Lq + t) * p.Hq + h) * p.D;
    for (int d = threadIdx.x; d < p.D; d += kThreads) {
        A v = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) v += part_o[w][d >> 2].v[d & 3];
        dst[d] = as_type<T>(L == A(0) ? A(0) : v / L);
    }
    if (threadIdx.x == 0) row_stats<A>(p, row, M, log2_any(L), L == A(0));
}

bool mma_fits(const Params& p, int dtype) {
    auto ok16 = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
    bool f = (dtype == NSC_F16 || dtype == NSC_BF16) && p.D % 8 == 0 && p.D <= 128 && ok16(p.k) &&
             ok16(p.v) && ok16(p.out) && (reinterpret_cast<uintptr_t>(p.q) & 3) == 0;
    for (int i = 0; i < 3; ++i)
        f = f && p.ks[i] % 8 == 0 && p.vs[i] % 8 == 0 && p.qs[i] % 2 == 0;
    return f;
}

bool f32_fits(const Params& p, int dtype) {
    auto ok16 = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
    bool f = dtype == NSC_F32 && p.D % 4 == 0 && p.D <= 128 && ok16(p.k) && ok16(p.v);
    for (int i = 0; i < 3; ++i) f = f && p.ks[i] % 4 == 0 && p.vs[i] % 4 == 0;
    return f;
}
// Rows of a block of decode_f32_kernel: eight fill the registers of two blocks an SM, and
// where a head has no more than four, three blocks keep more loads in flight.
int f32_rows(const Params& p) { return p.G * p.Lq > 4 ? 8 : 4; }

// Rows of a tensor-core block: two tiles of 16 where a head has more than one.
int mma_rows(const Params& p) { return p.G * p.Lq > 16 ? 32 : 16; }

// The cut of the long axis: one round of the blocks that fit the GPU at once (a
// block starts and ends with some thousand instructions a warp, the work of about
// a hundred keys, so two rounds of half the length cost more: 47 against 38 us for two
// caches of 65530 keys and 32 rows); at least 128 keys and 16 a row, so that a
// block's fixed cost (a few microseconds) and its parts are small beside its
// reads; at most 1024, which keeps the blocks of a large ragged batch even.
Split split_of(const Params& p, int rows_a_block) {
    Split s{};
    s.groups = (p.G * p.Lq + rows_a_block - 1) / rows_a_block;
    const int64_t units = static_cast<int64_t>(p.B) * p.Hkv * s.groups;
    const int64_t fit = 148 * (p.D <= 64 ? 3 : 2);
    const int64_t least = rows_a_block > 16 ? 320 : 128;
    int64_t c = (units * p.Lk + fit - 1) / fit;
    c = (c + 63) / 64 * 64;
    s.chunk = static_cast<int>(c < least ? least : (c > 1024 ? 1024 : c));
    s.n_chunk = p.Lk > 0 ? (p.Lk + s.chunk - 1) / s.chunk : 1;
    return s;
}

int64_t part_bytes(const Params& p, const Split& s, int dtype) {
    if (s.n_chunk == 1) return 0;
    return static_cast<int64_t>(p.B) * p.Hq * p.Lq * s.n_chunk * (part_wide(p.D) + 2) *
           (dtype == NSC_F64 ? 8 : 4);
}

template <typename T, int DP, int MT, bool CAP, bool BIAS>
nsc_status launch_mma(const Params& p, const Split& s, unsigned blocks, cudaStream_t st) {
    // 104 KB a block at DP = 128, 73 KB at 64
    constexpr int NS = DP == 64 ? 4 : 3, LD = 2 * DP + 16;
    auto kern = decode_mma_kernel<T, DP, MT, NS, CAP, BIAS>;
    const int ring = kWarps * NS * 2 * 16 * LD + (MT > 1 ? 16 * MT * LD : 0);
    const int heads = p.G < 16 * MT ? p.G : 16 * MT;
    const int smem = ring + (BIAS ? 4 * heads * p.nb + p.reach + 1 : 0);
    const nsc_status ready =
        raise_shared("token_attention_decode", reinterpret_cast<const void*>(kern), smem);
    if (ready != NSC_OK) return ready;
    kern<<<blocks, kMmaThreads, smem, st>>>(p, s);
    return check_launch("token_attention_decode");
}
template <typename T, int DP, int MT>
nsc_status run_mma_rows(const Params& p, const Split& s, unsigned blocks, cudaStream_t st) {
    if (p.cap > 0)
        return p.table ? launch_mma<T, DP, MT, true, true>(p, s, blocks, st)
                       : launch_mma<T, DP, MT, true, false>(p, s, blocks, st);
    return p.table ? launch_mma<T, DP, MT, false, true>(p, s, blocks, st)
                   : launch_mma<T, DP, MT, false, false>(p, s, blocks, st);
}
template <typename T, int DP>
nsc_status run_mma(const Params& p, const Split& s, unsigned blocks, cudaStream_t st) {
    return mma_rows(p) == 32 ? run_mma_rows<T, DP, 2>(p, s, blocks, st)
                             : run_mma_rows<T, DP, 1>(p, s, blocks, st);
}

template <typename T, typename A>
nsc_status run_any(const Params& p, const Split& s, unsigned blocks, cudaStream_t st) {
    const size_t smem = AnyShape<T, A>::smem(p.D);
    auto kern = decode_any_kernel<T, A>;
    const nsc_status ready =
        raise_shared("token_attention_decode", reinterpret_cast<const void*>(kern), smem);
    if (ready != NSC_OK) return ready;
    kern<<<blocks, kThreads, smem, st>>>(p, s);
    return check_launch("token_attention_decode");
}

template <int RB>
nsc_status run_f32(const Params& p, const Split& s, unsigned blocks, cudaStream_t st) {
    auto kern = p.D <= 32   ? decode_f32_kernel<32, RB>
                : p.D <= 64 ? decode_f32_kernel<64, RB>
                            : decode_f32_kernel<128, RB>;
    kern<<<blocks, kF32Threads, 0, st>>>(p, s);
    return check_launch("token_attention_decode");
}

// The join is launched before the chunks are done and its blocks start as the last of theirs
// ends (none triggers it earlier): what is hidden is the launch's latency.
template <typename T, typename A>
nsc_status launch_join(const Params& p, const Split& s, cudaStream_t st) {
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(p.B) * p.Hq * p.Lq));
    c.blockDim = dim3(kThreads);
    c.stream = st;
    c.attrs = &at;
    c.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&c, decode_join_kernel<T, A>, p, s);
    if (e != cudaSuccess)
        return fail(NSC_ERR_LAUNCH_FAILED, "token_attention_decode: %s", cudaGetErrorString(e));
    return check_launch("token_attention_decode");
}

}  // namespace

int64_t decode_workspace(const Params& p, int dtype) {
    // whichever kernel the call will take
    const int64_t a = part_bytes(p, split_of(p, mma_rows(p)), dtype);
    const int64_t b = part_bytes(p, split_of(p, kAnyRows), dtype);
    const int64_t c = part_bytes(p, split_of(p, f32_rows(p)), dtype);
    return std::max(a, std::max(b, c));
}

nsc_status decode(const Params& p, void* workspace, int dtype, cudaStream_t st) {
    const bool mma = mma_fits(p, dtype), f32 = f32_fits(p, dtype);
    Split s = split_of(p, mma ? mma_rows(p) : f32 ? f32_rows(p) : kAnyRows);
    s.part = workspace;
    if (s.n_chunk > 1 && !workspace)
        return fail(NSC_ERR_INVALID_ARG, "token_attention_decode: NULL pointer");
    const int64_t blocks = static_cast<int64_t>(p.B) * p.Hkv * s.groups * s.n_chunk;
    // (the join has a block a row)
    if (blocks >= (1LL << 31) || static_cast<int64_t>(p.B) * p.Hq * p.Lq >= (1LL << 31))
        return fail(NSC_ERR_INVALID_ARG, "token_attention_decode: too many tokens");
    const unsigned nb = static_cast<unsigned>(blocks);
    nsc_status r;
    if (mma && dtype == NSC_BF16)
        r = p.D <= 64 ? run_mma<__nv_bfloat16, 64>(p, s, nb, st)
                      : run_mma<__nv_bfloat16, 128>(p, s, nb, st);
    else if (mma)
        r = p.D <= 64 ? run_mma<__half, 64>(p, s, nb, st) : run_mma<__half, 128>(p, s, nb, st);
    else if (f32) r = f32_rows(p) == 8 ? run_f32<8>(p, s, nb, st) : run_f32<4>(p, s, nb, st);
    else if (dtype == NSC_F16) r = run_any<__half, float>(p, s, nb, st);
    else if (dtype == NSC_BF16) r = run_any<__nv_bfloat16, float>(p, s, nb, st);
    else if (dtype == NSC_F32) r = run_any<float, float>(p, s, nb, st);
    else r = run_any<double, double>(p, s, nb, st);
    if (r != NSC_OK || s.n_chunk == 1) return r;
    switch (dtype) {
        case NSC_F16: return launch_join<__half, float>(p, s, st);
        case NSC_BF16: return launch_join<__nv_bfloat16, float>(p, s, st);
        case NSC_F32: return launch_join<float, float>(p, s, st);
        default: return launch_join<double, double>(p, s, st);
    }
}

}  // namespace tok
}  // namespace nsc
