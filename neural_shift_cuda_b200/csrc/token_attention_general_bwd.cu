// token_attention_general_bwd.cu -- backward of token attention for every
// type, stride and head width, and the two small kernels around every
// backward pass (see token_attention_general.cuh).
//
// With P the softmax weights, dP = dO V^T and delta_i = sum_d dO_id O_id - dlse_i:
//     dz = P (dP - delta)                       (gradient at the biased score)
//     dtable[u] = sum of dz over the pairs whose distance is in bucket u
//     ds = dz (1 - tanh^2) scale                (gradient at q.k)
//     dQ = ds K,   dK = ds^T Q,   dV = P^T dO
// Two kernels, one with a query tile in place (dQ, table) and one with a key
// tile in place (dK, dV, summed over the query heads that share the key
// head).  Each recomputes the scores.  Where there are few tiles a cluster of blocks
// shares one: each takes every `share`-th step, and the sums are joined over the
// cluster's shared memory in the order of its ranks; no atomics, one order of every sum.
#include <climits>

#include "token_attention_general.cuh"

namespace nsc {
namespace tok {
namespace {

// The softmax weight and score gradients of one pair: s2 = unit x + bias with
// x the product, or its tanh; m and ll are the forward's row statistics.
template <typename A> struct Pair { A p, dz, ds; };

template <typename A>
__device__ __forceinline__ Pair<A> pair_grad(A dot, A dp, A bias, A m, A ll, A delta, bool seen,
                                             A scale, A unit, bool capped, A y1) {
    Pair<A> r{0, 0, 0};
    if (!seen || m == ninf<A>()) return r;
    A x = dot, slope = scale;
    if (capped) {
        x = tanh_(dot * y1);
        slope = scale * (1 - x * x);
    }
    r.p = exp2_(x * unit + bias - m - ll);
    r.dz = r.p * (dp - delta);
    r.ds = r.dz * slope;
    return r;
}

__device__ __forceinline__ uint32_t shared_at(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
// A thread's sums into a tile of shared memory, and those of every block of the
// cluster, row by row, out of it: block `rank` takes every `share`-th element.
template <typename A, int DP, int TL>
__device__ __forceinline__ void spill_tile(A* tile, const A (&v)[TL / 16][GenTile<DP, TL>::NG]
                                                             [GenTile<DP, TL>::VEC],
                                           int tx, int ty) {
    using G = GenTile<DP, TL>;
#pragma unroll
    for (int i = 0; i < G::MI; ++i)
#pragma unroll
        for (int g = 0; g < G::NG; ++g)
#pragma unroll
            for (int e = 0; e < G::VEC; ++e)
                tile[(ty + 16 * i) * G::LD + (g * 16 + tx) * G::VEC + e] = v[i][g][e];
}
template <typename A, int DP, int TL, typename F>
__device__ __forceinline__ void join_tile(const A* tile, int rank, int share, int D, F put) {
    using G = GenTile<DP, TL>;
    for (int i = threadIdx.x * share + rank; i < TL * DP; i += kGenThreads * share) {
        const int r = i / DP, d = i % DP;
        if (d >= D) continue;
        A v = 0;
        for (int x = 0; x < share; ++x) v += cluster_load<A>(shared_at(tile + r * G::LD + d), x);
        put(r, d, v);
    }
}

template <typename T, typename A, int DP, int TL>
__global__ __launch_bounds__(kGenThreads) void general_dq_kernel(Params p, Grads gr, int share) {
    using G = GenTile<DP, TL>;
    constexpr int MI = G::MI;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ int box[2];
    __shared__ A diag[2 * TL], mines[kGenThreads];
    A* Qs = reinterpret_cast<A*>(smem_raw);
    A* Os = Qs + TL * G::LD;
    A* Ks = Os + TL * G::LD;
    A* Vs = Ks + TL * G::LD;
    A* Ps = Vs + TL * G::LD;
    A* bias = Ps + TL * G::LP;

    const int nt = (p.Lq + TL - 1) / TL;
    const int64_t BH = static_cast<int64_t>(p.B) * p.Hq;
    const int64_t id = blockIdx.x / share;
    const int rank = static_cast<int>(blockIdx.x % share);
    const int t = nt - 1 - static_cast<int>(id / BH);
    const int bh = static_cast<int>(id % BH), b = bh / p.Hq, h = bh % p.Hq;
    const int hk = h / p.G, q0 = t * TL, off = p.Lk - p.Lq;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[2];
    const T* go = static_cast<const T*>(gr.dout) + b * gr.dos[0] + h * gr.dos[2];
    const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
    const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];

    int lo[MI], hi[MI], slo = INT_MAX, shi = 0;
    A m[MI], ll[MI], delta[MI];
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int row = q0 + ty + 16 * i;
        lo[i] = hi[i] = 0;
        m[i] = ll[i] = delta[i] = 0;
        if (row < p.Lq) {
            key_span(p, b, row, p.Lk, lo[i], hi[i]);
            const int64_t at = static_cast<int64_t>(bh) * p.Lq + row;
            m[i] = static_cast<const A*>(p.stats)[at];
            ll[i] = static_cast<const A*>(p.stats)[BH * p.Lq + at];
            delta[i] = static_cast<const A*>(gr.delta)[at];
        }
        if (hi[i] > lo[i]) { slo = min(slo, lo[i]); shi = max(shi, hi[i]); }
    }
    int first, last;
    join_spans(slo, shi, box, first, last);
    if (p.table) load_bias<A>(p, h, bias);
    load_tile<T, A, DP, TL>(Qs, q, p.qs[1], q0, 0, p.Lq, p.D);
    load_tile<T, A, DP, TL>(Os, go, gr.dos[1], q0, 0, p.Lq, p.D);

    A dq[MI][G::NG][G::VEC];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int g = 0; g < G::NG; ++g)
#pragma unroll
            for (int e = 0; e < G::VEC; ++e) dq[i][g][e] = 0;
    A mine = 0;  // bucket threadIdx.x of the table gradient
    const A scale = p.scale, unit = (p.cap > 0 ? p.cap : p.scale) * kLog2e;
    const A y1 = p.cap > 0 ? p.scale / p.cap : 0;
    for (int k0 = (first / TL + rank) * TL; k0 < last; k0 += TL * share) {
        __syncthreads();
        const bool odd = load_tile<T, A, DP, TL>(Ks, k, p.ks[1], k0, first, last, p.D);
        load_tile<T, A, DP, TL>(Vs, v, p.vs[1], k0, first, last, p.D);
        const bool strict = __syncthreads_or(odd);
        A s[MI][MI], dp[MI][MI];
        dot_tile<A, DP, TL>(Qs, Ks, tx, ty, s);
        dot_tile<A, DP, TL>(Os, Vs, tx, ty, dp);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < MI; ++j) {
                const int key = k0 + tx + 16 * j;
                const A bi = p.table ? bias[distance_at(p, key - (q0 + ty + 16 * i + off))] : A(0);
                const Pair<A> r = pair_grad<A>(s[i][j], dp[i][j], bi, m[i], ll[i], delta[i],
                                               key >= lo[i] && key < hi[i], scale, unit, p.cap > 0, y1);
                s[i][j] = r.ds;
                Ps[(ty + 16 * i) * G::LP + tx + 16 * j] = gr.tab ? r.dz : r.ds;
            }
        __syncthreads();
        if (gr.tab) {
            // sums along the diagonals of the tile, then over the distances
            // of each bucket, both in a fixed order
            if (threadIdx.x < 2 * TL - 1) {
                const int dd = static_cast<int>(threadIdx.x) - (TL - 1);
                A sum = 0;
                for (int r = max(0, -dd); r < min(TL, TL - dd); ++r) sum += Ps[r * G::LP + r + dd];
                diag[threadIdx.x] = sum;
            }
            __syncthreads();
            if (threadIdx.x < p.nb) {
                const int rel0 = k0 - (q0 + off) - (TL - 1);
                A part = 0;   // a tile's share first: shorter chains of rounded sums
                for (int i = 0; i < 2 * TL - 1; ++i) {
                    const int u = __ldg(p.lut + distance_at(p, rel0 + i));
                    if (min(max(u, 0), p.nb - 1) == static_cast<int>(threadIdx.x)) part += diag[i];
                }
                mine += part;
            }
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < MI; ++j)
                    Ps[(ty + 16 * i) * G::LP + tx + 16 * j] = s[i][j];
            __syncthreads();
        }
        mix_tile<A, DP, TL>(Ps, Ks, tx, ty, strict, dq);
    }
    if (share > 1) {
        __syncthreads();
        spill_tile<A, DP, TL>(Qs, dq, tx, ty);
        mines[threadIdx.x] = mine;
        cluster_sync();
        join_tile<A, DP, TL>(Qs, rank, share, p.D, [&](int r, int d, A v) {
            if (q0 + r < p.Lq)
                static_cast<T*>(gr.dq)[((static_cast<int64_t>(b) * p.Lq + q0 + r) * p.Hq + h) * p.D + d] =
                    store_as<T>(v);
        });
        if (rank == 0 && gr.tab)
            for (int r = 1; r < share; ++r) mine += cluster_load<A>(shared_at(mines + threadIdx.x), r);
        cluster_sync();   // no block leaves while another reads its memory
        if (rank) return;
    } else {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int row = q0 + ty + 16 * i;
            if (row >= p.Lq) continue;
            T* dst = static_cast<T*>(gr.dq) +
                     ((static_cast<int64_t>(b) * p.Lq + row) * p.Hq + h) * p.D;
#pragma unroll
            for (int g = 0; g < G::NG; ++g)
#pragma unroll
                for (int e = 0; e < G::VEC; ++e) {
                    const int d = (g * 16 + tx) * G::VEC + e;
                    if (d < p.D) dst[d] = store_as<T>(dq[i][g][e]);
                }
        }
    }
    if (gr.tab && threadIdx.x < p.nb)
        static_cast<A*>(gr.tab)[(static_cast<int64_t>(h) * gr.n_part + b * nt + t) * p.nb +
                                threadIdx.x] = mine;
}

template <typename T, typename A, int DP, int TL>
__global__ __launch_bounds__(kGenThreads) void general_dkv_kernel(Params p, Grads gr, int share) {
    using G = GenTile<DP, TL>;
    constexpr int MI = G::MI;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ int box[2];
    __shared__ A ms[TL], lls[TL], deltas[TL];
    A* Ks = reinterpret_cast<A*>(smem_raw);
    A* Vs = Ks + TL * G::LD;
    A* Qs = Vs + TL * G::LD;
    A* Os = Qs + TL * G::LD;
    A* Ps = Os + TL * G::LD;   // P^T, keys by queries
    A* Ss = Ps + TL * G::LP;   // ds^T
    A* bias = Ss + TL * G::LP;

    const int64_t BH = static_cast<int64_t>(p.B) * p.Hkv;
    const int64_t id = blockIdx.x / share;
    const int rank = static_cast<int>(blockIdx.x % share);
    const int t = static_cast<int>(id / BH);
    const int bh = static_cast<int>(id % BH), b = bh / p.Hkv, hk = bh % p.Hkv;
    const int k0 = t * TL, off = p.Lk - p.Lq;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
    const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];

    int lo[MI], hi[MI], slo = INT_MAX, shi = 0;
#pragma unroll
    for (int j = 0; j < MI; ++j) {
        query_span(p, b, k0 + tx + 16 * j, lo[j], hi[j]);
        if (hi[j] > lo[j]) { slo = min(slo, lo[j]); shi = max(shi, hi[j]); }
    }
    int first, last;
    join_spans(slo, shi, box, first, last);
    load_tile<T, A, DP, TL>(Ks, k, p.ks[1], k0, 0, p.Lk, p.D);
    load_tile<T, A, DP, TL>(Vs, v, p.vs[1], k0, 0, p.Lk, p.D);

    A dk[MI][G::NG][G::VEC], dv[MI][G::NG][G::VEC];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int g = 0; g < G::NG; ++g)
#pragma unroll
            for (int e = 0; e < G::VEC; ++e) dk[i][g][e] = dv[i][g][e] = 0;
    const A scale = p.scale, unit = (p.cap > 0 ? p.cap : p.scale) * kLog2e;
    const A y1 = p.cap > 0 ? p.scale / p.cap : 0;
    int step = 0;
    for (int u = 0; u < p.G; ++u) {
        const int h = hk * p.G + u;
        const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[2];
        const T* go = static_cast<const T*>(gr.dout) + b * gr.dos[0] + h * gr.dos[2];
        const int64_t row0 = (static_cast<int64_t>(b) * p.Hq + h) * p.Lq;
        __syncthreads();
        if (p.table) load_bias<A>(p, h, bias);
        for (int q0 = first / TL * TL; q0 < last; q0 += TL, ++step) {
            if (step % share != rank) continue;
            __syncthreads();
            bool odd = load_tile<T, A, DP, TL>(Qs, q, p.qs[1], q0, first, last, p.D);
            odd |= load_tile<T, A, DP, TL>(Os, go, gr.dos[1], q0, first, last, p.D);
            if (threadIdx.x < TL) {
                const int row = q0 + threadIdx.x;
                const int64_t rows = static_cast<int64_t>(p.B) * p.Hq * p.Lq;
                ms[threadIdx.x] = row < p.Lq ? static_cast<const A*>(p.stats)[row0 + row] : 0;
                lls[threadIdx.x] =
                    row < p.Lq ? static_cast<const A*>(p.stats)[rows + row0 + row] : 0;
                deltas[threadIdx.x] =
                    row < p.Lq ? static_cast<const A*>(gr.delta)[row0 + row] : 0;
            }
            const bool strict = __syncthreads_or(odd);
            A s[MI][MI], dp[MI][MI];
            dot_tile<A, DP, TL>(Qs, Ks, tx, ty, s);
            dot_tile<A, DP, TL>(Os, Vs, tx, ty, dp);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < MI; ++j) {
                    const int r = ty + 16 * i, c = tx + 16 * j, row = q0 + r;
                    const A bi = p.table ? bias[distance_at(p, k0 + c - (row + off))] : A(0);
                    const Pair<A> g = pair_grad<A>(s[i][j], dp[i][j], bi, ms[r], lls[r], deltas[r],
                                                   row >= lo[j] && row < hi[j], scale, unit, p.cap > 0, y1);
                    Ps[c * G::LP + r] = g.p;
                    Ss[c * G::LP + r] = g.ds;
                }
            __syncthreads();
            mix_tile<A, DP, TL>(Ps, Os, tx, ty, strict, dv);
            mix_tile<A, DP, TL>(Ss, Qs, tx, ty, strict, dk);
        }
    }
    if (share > 1) {
        __syncthreads();
        spill_tile<A, DP, TL>(Qs, dk, tx, ty);
        spill_tile<A, DP, TL>(Os, dv, tx, ty);
        cluster_sync();
        auto put = [&](void* out) {
            return [&, out](int r, int d, A v) {
                if (k0 + r < p.Lk)
                    static_cast<T*>(out)[((static_cast<int64_t>(b) * p.Lk + k0 + r) * p.Hkv + hk) * p.D +
                                         d] = store_as<T>(v);
            };
        };
        join_tile<A, DP, TL>(Qs, rank, share, p.D, put(gr.dk));
        join_tile<A, DP, TL>(Os, rank, share, p.D, put(gr.dv));
        cluster_sync();   // no block leaves while another reads its memory
        return;
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int row = k0 + ty + 16 * i;
        if (row >= p.Lk) continue;
        const int64_t at = ((static_cast<int64_t>(b) * p.Lk + row) * p.Hkv + hk) * p.D;
#pragma unroll
        for (int g = 0; g < G::NG; ++g)
#pragma unroll
            for (int e = 0; e < G::VEC; ++e) {
                const int d = (g * 16 + tx) * G::VEC + e;
                if (d >= p.D) continue;
                static_cast<T*>(gr.dk)[at + d] = store_as<T>(dk[i][g][e]);
                static_cast<T*>(gr.dv)[at + d] = store_as<T>(dv[i][g][e]);
            }
    }
}

// delta: one warp per (token, head) of the contiguous out.
template <typename T, typename A>
__global__ __launch_bounds__(256) void delta_kernel(Params p, Grads gr) {
    const int64_t n = static_cast<int64_t>(p.B) * p.Lq * p.Hq;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (w >= n) return;
    const int lane = threadIdx.x & 31;
    const int h = static_cast<int>(w % p.Hq);
    const int64_t bl = w / p.Hq, b = bl / p.Lq, l = bl % p.Lq;
    const T* o = static_cast<const T*>(p.out) + w * p.D;
    const T* lo = p.residue ? static_cast<const T*>(p.residue) + w * p.D : nullptr;
    const T* g = static_cast<const T*>(gr.dout) + b * gr.dos[0] + l * gr.dos[1] + h * gr.dos[2];
    A sum = 0;
    for (int d = lane; d < p.D; d += 32) {
        A x = to_acc(o[d]);
        if (lo) x += to_acc(lo[d]);
        sum += x * static_cast<A>(to_acc(g[d]));
    }
#pragma unroll
    for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    if (lane == 0) {
        const int64_t at = (b * p.Hq + h) * p.Lq + l;
        if (gr.dlse) sum -= static_cast<const A*>(gr.dlse)[at];
        static_cast<A*>(gr.delta)[at] = sum;
    }
}

// One block per table entry: the partial sums of its head and bucket.
template <typename A, typename O>
__global__ __launch_bounds__(256) void table_join_kernel(const A* tab, O* out, int Hq, int n_part,
                                                         int nb) {
    __shared__ double part[8];
    const int h = blockIdx.x % Hq, u = blockIdx.x / Hq;
    double sum = 0;
    for (int i = threadIdx.x; i < n_part; i += 256)
        sum += tab[(static_cast<int64_t>(h) * n_part + i) * nb + u];
#pragma unroll
    for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    for (int i = 1; i < 8; ++i) sum += part[i];
    if constexpr (sizeof(O) == 8) out[static_cast<int64_t>(u) * Hq + h] = sum;
    else out[static_cast<int64_t>(u) * Hq + h] = from_float<O>(static_cast<float>(sum));
}

template <typename T, typename A, int DP, int TL>
nsc_status launch(const Params& p, const Grads& g, cudaStream_t st) {
    const int extra = p.table ? 2 * p.reach + 1 : 0;
    const size_t smq = gen_smem<A, DP, TL>(4, 1, extra), smk = gen_smem<A, DP, TL>(4, 2, extra);
    auto kq = general_dq_kernel<T, A, DP, TL>;
    auto kk = general_dkv_kernel<T, A, DP, TL>;
    const char* op = "token_attention backward";
    nsc_status r = raise_shared(op, reinterpret_cast<const void*>(kq), smq);
    if (r == NSC_OK) r = raise_shared(op, reinterpret_cast<const void*>(kk), smk);
    if (r != NSC_OK) return r;
    const int64_t nq = static_cast<int64_t>((p.Lq + TL - 1) / TL) * p.B * p.Hq;
    const int64_t nk = static_cast<int64_t>((p.Lk + TL - 1) / TL) * p.B * p.Hkv;
    // blocks of a tile: up to about four an SM in all, none without a step
    auto share_of = [](int64_t tiles, int64_t steps) {
        int n = 1;
        while (n < 8 && tiles * n * 2 <= 4 * 148 && n * 2 <= steps) n *= 2;
        return n;
    };
    const int nqt = (p.Lq + TL - 1) / TL, nkt = (p.Lk + TL - 1) / TL;
    const int sk = share_of(nk, static_cast<int64_t>(p.G) * nqt), sq = share_of(nq, nkt);
    if (nk && g.dk) r = launch_cluster(op, kk, nk * sk, kGenThreads, smk, sk, st, p, g, sk);
    if (r == NSC_OK && nq && g.dq) r = launch_cluster(op, kq, nq * sq, kGenThreads, smq, sq, st, p, g, sq);
    if (r != NSC_OK) return r;
    return check_launch("token_attention backward");
}

}  // namespace

nsc_status general_bwd(const Params& p, const Grads& g, int dtype, cudaStream_t st) {
#define NSC_GEN_ARGS p, g, st
    NSC_GEN_DISPATCH(launch)
#undef NSC_GEN_ARGS
}

nsc_status launch_delta(const Params& p, const Grads& g, int dtype, cudaStream_t st) {
    const int64_t n = (static_cast<int64_t>(p.B) * p.Lq * p.Hq + 7) / 8;
    const unsigned blocks = static_cast<unsigned>(n);
    if (!blocks) return ok();
    switch (dtype) {
        case NSC_F16: delta_kernel<__half, float><<<blocks, 256, 0, st>>>(p, g); break;
        case NSC_BF16: delta_kernel<__nv_bfloat16, float><<<blocks, 256, 0, st>>>(p, g); break;
        case NSC_F32: delta_kernel<float, float><<<blocks, 256, 0, st>>>(p, g); break;
        default: delta_kernel<double, double><<<blocks, 256, 0, st>>>(p, g);
    }
    return check_launch("token_attention backward");
}

nsc_status launch_table_join(const Params& p, const Grads& g, void* out, cudaStream_t st) {
    const unsigned blocks = static_cast<unsigned>(p.Hq) * p.nb;
    const float* tab = static_cast<const float*>(g.tab);
    switch (p.table_dtype) {
        case NSC_F16:
            table_join_kernel<<<blocks, 256, 0, st>>>(tab, static_cast<__half*>(out), p.Hq,
                                                      g.n_part, p.nb);
            break;
        case NSC_BF16:
            table_join_kernel<<<blocks, 256, 0, st>>>(tab, static_cast<__nv_bfloat16*>(out), p.Hq,
                                                      g.n_part, p.nb);
            break;
        case NSC_F32:
            table_join_kernel<<<blocks, 256, 0, st>>>(tab, static_cast<float*>(out), p.Hq,
                                                      g.n_part, p.nb);
            break;
        default:
            table_join_kernel<<<blocks, 256, 0, st>>>(static_cast<const double*>(g.tab),
                                                      static_cast<double*>(out), p.Hq, g.n_part,
                                                      p.nb);
    }
    return check_launch("token_attention backward");
}

}  // namespace tok
}  // namespace nsc
