// token_attention_general_fwd.cu -- forward of token attention for every
// type, stride and head width (see token_attention_general.cuh).
//
// One block per (query tile, head, batch entry).  Keys pass tile by tile with
// the running maximum and sum of a softmax: when the maximum m of a row moves
// to m', its sum and its output row are scaled by 2^(m - m').
#include <climits>

#include "token_attention_general.cuh"

namespace nsc {
namespace tok {
namespace {

template <typename T, typename A, int DP, int TL>
__global__ __launch_bounds__(kGenThreads) void general_fwd_kernel(Params p) {
    using G = GenTile<DP, TL>;
    constexpr int MI = G::MI;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ int box[2];
    A* Qs = reinterpret_cast<A*>(smem_raw);
    A* Ks = Qs + TL * G::LD;
    A* Vs = Ks + TL * G::LD;
    A* Ps = Vs + TL * G::LD;
    A* bias = Ps + TL * G::LP;

    const int nt = (p.Lq + TL - 1) / TL;
    const int64_t BH = static_cast<int64_t>(p.B) * p.Hq;
    // late query tiles first: under a causal mask they see the most keys
    const int t = nt - 1 - static_cast<int>(blockIdx.x / BH);
    const int bh = static_cast<int>(blockIdx.x % BH), b = bh / p.Hq, h = bh % p.Hq;
    const int hk = h / p.G, n = keys_of(p, b), q0 = t * TL;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[2];
    const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
    const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];

    int lo[MI], hi[MI], slo = INT_MAX, shi = 0;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int row = q0 + ty + 16 * i;
        lo[i] = hi[i] = 0;
        if (row < p.Lq) key_span(p, b, row, n, lo[i], hi[i]);
        if (hi[i] > lo[i]) { slo = min(slo, lo[i]); shi = max(shi, hi[i]); }
    }
    int first, last;
    join_spans(slo, shi, box, first, last);
    if (p.table) load_bias<A>(p, h, bias);
    load_tile<T, A, DP, TL>(Qs, q, p.qs[1], q0, 0, p.Lq, p.D);

    A m[MI], l[MI], o[MI][G::NG][G::VEC];
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        m[i] = ninf<A>();
        l[i] = 0;
#pragma unroll
        for (int g = 0; g < G::NG; ++g)
#pragma unroll
            for (int e = 0; e < G::VEC; ++e) o[i][g][e] = 0;
    }
    const A unit = (p.cap > 0 ? p.cap : p.scale) * kLog2e, y1 = p.cap > 0 ? p.scale / p.cap : 0;
    for (int k0 = first / TL * TL; k0 < last; k0 += TL) {
        __syncthreads();
        load_tile<T, A, DP, TL>(Ks, k, p.ks[1], k0, first, last, p.D);
        const bool odd = load_tile<T, A, DP, TL>(Vs, v, p.vs[1], k0, first, last, p.D);
        const bool strict = __syncthreads_or(odd);
        A s[MI][MI];
        dot_tile<A, DP, TL>(Qs, Ks, tx, ty, s);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int rel0 = k0 + tx - (q0 + ty + 16 * i + n - p.Lq);
            A top = ninf<A>();
#pragma unroll
            for (int j = 0; j < MI; ++j) {
                const int key = k0 + tx + 16 * j;
                A x = (p.cap > 0 ? tanh_(s[i][j] * y1) : s[i][j]) * unit;
                if (p.table) x += bias[distance_at(p, rel0 + 16 * j)];
                s[i][j] = key >= lo[i] && key < hi[i] ? x : ninf<A>();
                top = s[i][j] > top || s[i][j] != s[i][j] ? s[i][j] : top;
            }
#pragma unroll
            for (int w = 1; w < 16; w <<= 1) {
                const A other = __shfl_xor_sync(0xffffffffu, top, w);
                top = other > top || other != other ? other : top;
            }
            const A mn = m[i] > top ? m[i] : top;
            const A ref = mn == ninf<A>() ? A(0) : mn;
            const A corr = exp2_(m[i] - ref);
            A sum = 0;
#pragma unroll
            for (int j = 0; j < MI; ++j) {
                const A e = exp2_(s[i][j] - ref);
                sum += e;
                Ps[(ty + 16 * i) * G::LP + tx + 16 * j] = e;
            }
#pragma unroll
            for (int w = 1; w < 16; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            l[i] = l[i] * corr + sum;
            m[i] = mn;
#pragma unroll
            for (int g = 0; g < G::NG; ++g)
#pragma unroll
                for (int e = 0; e < G::VEC; ++e) o[i][g][e] *= corr;
        }
        __syncthreads();
        mix_tile<A, DP, TL>(Ps, Vs, tx, ty, strict, o);
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int row = q0 + ty + 16 * i;
        if (row >= p.Lq) continue;
        const A inv = l[i] == A(0) ? A(0) : 1 / l[i];
        const int64_t at = ((static_cast<int64_t>(b) * p.Lq + row) * p.Hq + h) * p.D;
        T* dst = static_cast<T*>(p.out) + at;
#pragma unroll
        for (int g = 0; g < G::NG; ++g)
#pragma unroll
            for (int e = 0; e < G::VEC; ++e) {
                const int d = (g * 16 + tx) * G::VEC + e;
                if (d >= p.D) continue;
                const A x = o[i][g][e] * inv;
                const T y = store_as<T>(x);
                dst[d] = y;
                if (p.residue) static_cast<T*>(p.residue)[at + d] = store_as<T>(x - to_acc(y));
            }
        if (tx == 0)
            row_stats<A>(p, static_cast<int64_t>(bh) * p.Lq + row, m[i], log2_(l[i]),
                         l[i] == A(0));
    }
}

template <typename T, typename A, int DP, int TL>
nsc_status launch(const Params& p, cudaStream_t st) {
    const int64_t blocks = static_cast<int64_t>((p.Lq + TL - 1) / TL) * p.B * p.Hq;
    const size_t smem = gen_smem<A, DP, TL>(3, 1, p.table ? 2 * p.reach + 1 : 0);
    auto kern = general_fwd_kernel<T, A, DP, TL>;
    const nsc_status ready = raise_shared("token_attention", reinterpret_cast<const void*>(kern), smem);
    if (ready != NSC_OK) return ready;
    kern<<<static_cast<unsigned>(blocks), kGenThreads, smem, st>>>(p);
    return check_launch("token_attention");
}

}  // namespace

// A tile of 64 reads shared memory half as often a product as one of 32, but where 64
// leaves fewer than two blocks an SM, 32 (four times the tiles) is faster: the kernels of
// a training step over 2 x 333 tokens, 4 heads of 64, fp32, 177 against 137 us.
int general_tile(int dtype, int64_t B, int64_t Hkv, int64_t Lq, int64_t Lk, int64_t D) {
    if (dtype == NSC_F64 || D > 128) return 32;
    return B * Hkv * (((Lq > Lk ? Lq : Lk) + 63) / 64) < 2 * 148 ? 32 : 64;
}

nsc_status general_fwd(const Params& p, int dtype, cudaStream_t st) {
#define NSC_GEN_ARGS p, st
    NSC_GEN_DISPATCH(launch)
#undef NSC_GEN_ARGS
}

}  // namespace tok
}  // namespace nsc
