// token_attention.h -- what the token-attention kernels share: the call's
// parameters as the kernels read them, the visible spans, and the launchers
// of the kernel families behind the entry points in token_attention.cu.
#pragma once

#include "nsc_host.h"

namespace nsc {
namespace tok {

struct Params {
    const void *q, *k, *v;
    int64_t qs[3], ks[3], vs[3];      // element strides of b, l, h
    void* out;                        // contiguous (B, Lq, Hq, D)
    void* lse;                        // contiguous (B, Hq, Lq), nullable
    void* stats;                      // (2, B, Hq, Lq), nullable: see row_stats
    void* residue;                    // like out, nullable: what rounding out dropped
    int B, Lq, Lk, Hq, Hkv, G, D;     // G = Hq / Hkv
    int causal;
    const int32_t *docs, *prefix, *lengths, *lut;
    int64_t docs_stride, prefix_stride;
    int n_docs, prefix_cols, nb, reach;
    const void* table;
    int table_dtype;
    double scale, cap;
};

struct Grads {
    const void *dout, *dlse;
    int64_t dos[3];
    void *dq, *dk, *dv;               // contiguous
    void *delta;                      // (B, Hq, Lq): sum_d dout out - dlse
    void* tab;                        // (Hq, n_part, nb) partial sums, or null
    int n_part;
    // fp16 on the tensor cores: norms of the value rows (B, Hkv, Lk), the largest that each
    // query sees (B, Hkv, Lq), and of each 128 query rows (B, Hq, .) the largest norm of dout
    // and largest |delta|
    const float *value_norms, *seen_norms, *row_norms, *row_deltas;
};

// Document [s, e) of position t: the last bound <= t opens it.  Bounds are
// clamped to [0, n], so no call reads past a tensor whatever they hold.
__device__ __forceinline__ bool find_doc(const Params& p, int b, int t, int n, int& s, int& e,
                                         int& doc) {
    const int32_t* d = p.docs + b * p.docs_stride;
    int lo = 0, hi = p.n_docs + 1;    // bounds [0, lo) are <= t, [hi, ...) are > t
    while (lo < hi) {
        const int m = (lo + hi) >> 1;
        if (__ldg(d + m) <= t) lo = m + 1; else hi = m;
    }
    doc = lo - 1;
    if (doc < 0 || doc >= p.n_docs) return false;
    s = min(max(__ldg(d + doc), 0), n);
    e = min(max(__ldg(d + doc + 1), 0), n);
    return true;
}

__device__ __forceinline__ int prefix_of(const Params& p, int b, int doc, int n) {
    if (!p.prefix) return 0;
    return min(max(__ldg(p.prefix + b * p.prefix_stride + doc), 0), n);
}

__device__ __forceinline__ int keys_of(const Params& p, int b) {
    return p.lengths ? min(max(__ldg(p.lengths + b), 0), p.Lk) : p.Lk;
}

// Every mask here is one interval of keys per query: keys [lo, hi) are
// visible to query i (hi <= lo: none).  n = keys_of(p, b).
__device__ __forceinline__ void key_span(const Params& p, int b, int i, int n, int& lo, int& hi) {
    const int pos = i + n - p.Lq;
    int s = 0, e = n, doc = 0;
    if (p.docs && !find_doc(p, b, pos, n, s, e, doc)) { lo = hi = 0; return; }
    lo = s;
    hi = p.causal ? min(e, max(pos + 1, s + prefix_of(p, b, doc, n))) : e;
}

// The same relation from a key: queries [lo, hi) see key j (lengths is null).
__device__ __forceinline__ void query_span(const Params& p, int b, int j, int& lo, int& hi) {
    const int off = p.Lk - p.Lq;
    int s = 0, e = p.Lk, doc = 0;
    if (j >= p.Lk || (p.docs && !find_doc(p, b, j, p.Lk, s, e, doc))) { lo = hi = 0; return; }
    const bool all = !p.causal || j < s + prefix_of(p, b, doc, p.Lk);
    lo = all ? (p.docs ? s : 0) : max(0, j - off);
    hi = p.docs ? e : p.Lq;
}

// Bias of bucket b for head h.
template <typename A>
__device__ __forceinline__ A table_at(const Params& p, int b, int h) {
    b = min(max(b, 0), p.nb - 1);
    const int64_t at = static_cast<int64_t>(b) * p.Hq + h;
    switch (p.table_dtype) {
        case NSC_F16: return __half2float(static_cast<const __half*>(p.table)[at]);
        case NSC_BF16: return __bfloat162float(static_cast<const __nv_bfloat16*>(p.table)[at]);
        case NSC_F32: return static_cast<const float*>(p.table)[at];
    }
    return static_cast<A>(static_cast<const double*>(p.table)[at]);
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                     : "memory");
}
// The value at this block's shared address `at`, in block `rank` of the cluster.
template <typename A> __device__ __forceinline__ A cluster_load(uint32_t at, int rank) {
    uint32_t a;
    A v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(at), "r"(rank));
    if constexpr (sizeof(A) == 4)
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    else
        asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(a) : "memory");
    return v;
}
// A launch of `blocks` blocks in clusters of `cluster`.
template <typename K, typename... Args>
inline nsc_status launch_cluster(const char* op, K kern, int64_t blocks, int threads, size_t smem,
                                 int cluster, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = static_cast<unsigned>(cluster);
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (e != cudaSuccess)
        return fail(NSC_ERR_LAUNCH_FAILED, "%s: kernel launch failed: %s", op, cudaGetErrorString(e));
    return ok();
}

constexpr double kLog2e = 1.4426950408889634;
constexpr double kLn2 = 0.6931471805599453;

// Scores are held in units of log 2, s2 = s log2(e).  A finite bias is kept
// within 1e37, so that the sum of a score and the lowest value of its type
// stays finite (and a row that sees nothing else has a uniform softmax).
template <typename A>
__device__ __forceinline__ A bias2_at(const Params& p, int b, int h) {
    const A t = table_at<A>(p, b, h);
    if (!(t - t == A(0))) return t;   // infinities and NaN as they are
    const A v = t * static_cast<A>(kLog2e);
    return v < A(-1e37) ? A(-1e37) : (v > A(1e37) ? A(1e37) : v);
}

// What a forward leaves for its backward: the reference m and log2 of the sum
// of 2^(s2 - m), apart (their sum would lose the sum's digits beside a large
// m).  A row that sees nothing has m = -inf.
template <typename A>
__device__ __forceinline__ void row_stats(const Params& p, int64_t row, A m, A log2_sum, bool none) {
    const int64_t n = static_cast<int64_t>(p.B) * p.Hq * p.Lq;
    if (p.stats) {
        static_cast<A*>(p.stats)[row] = none ? A(-INFINITY) : m;
        static_cast<A*>(p.stats)[n + row] = none ? A(0) : log2_sum;
    }
    if (p.lse)
        static_cast<A*>(p.lse)[row] =
            none ? A(-INFINITY) : m * static_cast<A>(kLn2) + log2_sum * static_cast<A>(kLn2);
}

// Kernels for any type, strides and head width (token_attention_general.cu).
nsc_status general_fwd(const Params& p, int dtype, cudaStream_t st);
nsc_status general_bwd(const Params& p, const Grads& g, int dtype, cudaStream_t st);
int general_tile(int dtype, int64_t B, int64_t Hkv, int64_t Lq, int64_t Lk, int64_t D);

// Tensor-core kernels for fp16 / bf16 (token_attention_tc_*.cu); tc_fits: whether a
// call's layout is one that their TMA boxes describe.
bool tc_fits(const Params& p, int dtype);
nsc_status tc_fwd(const Params& p, int dtype, cudaStream_t st);
// token_attention_short.cu
bool short_fits(const Params& p, int dtype);
nsc_status short_fwd(const Params& p, int dtype, cudaStream_t st);
bool tc_bwd_fits(const Params& p, const Grads& g, int dtype);
int64_t tc_bwd_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t Lq, int64_t Lk,
                         int64_t n_buckets);
nsc_status tc_bwd(const Params& p, Grads g, void* workspace, void* grad_table, int dtype,
                  cudaStream_t st);

// token_decode.cu
int64_t decode_workspace(const Params& p, int dtype);
nsc_status decode(const Params& p, void* workspace, int dtype, cudaStream_t st);

// delta (and its layout (B, Hq, Lq)) for a backward pass; joining of the
// table-gradient partials.
nsc_status launch_delta(const Params& p, const Grads& g, int dtype, cudaStream_t st);
nsc_status launch_table_join(const Params& p, const Grads& g, void* grad_table, cudaStream_t st);

}  // namespace tok
}  // namespace nsc
