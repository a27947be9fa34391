// token_attention_tc.cu -- host side of the tensor-core token-attention kernels:
// which calls they take, tensor maps, shared-memory and register checks.
#include <cudaTypedefs.h>

#include <cmath>

#include "token_attention_tc.cuh"

namespace nsc {
namespace tok {
namespace {

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) !=
                cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    return fn;
}

// The row records, LN lanes a row, 16 bytes a lane, four rows of a lane in flight.  Bound
// by memory: out, residue and grad_out read once (4 x 2048 tokens, 16 heads of 64: 11 us
// for 50 MB, 4.6 TB/s; with one row in flight and half the lanes idle 19 us).
// TOPS (fp16, for the scales of the score gradients): and the largest norm and |delta| of each
// block's rows.  A row that is not finite does not set them: what sees it is NaN anyway.
// (Eight blocks an SM, 32 registers: with 34 it took 26 us for 20, 8192 tokens, 16 heads of 128.)
template <typename T, int LN, bool TOPS>
__global__ __launch_bounds__(256, 8) void record_kernel(Params p, Grads g, RowRec* recs, float* norms,
                                                     float* deltas, int blocks_h) {
    constexpr int RB = 256 / LN;   // rows side by side
    __shared__ float top[2][RB];
    const int bh = blockIdx.x / blocks_h, blk = blockIdx.x % blocks_h;
    const int b = bh / p.Hq, h = bh % p.Hq, sub = threadIdx.x / LN, c = threadIdx.x % LN;
    const int64_t rows = static_cast<int64_t>(p.B) * p.Hq * p.Lq;
    float most = 0.f, most_delta = 0.f;
#pragma unroll 4
    for (int u = 0; u < kRecRows / RB; ++u) {
        const int l = blk * kRecRows + RB * u + sub;
        float sum = 0.f, sq = 0.f;
        if (l < p.Lq && 8 * c < p.D) {
            const int64_t at = ((static_cast<int64_t>(b) * p.Lq + l) * p.Hq + h) * p.D + 8 * c;
            const uint4 o = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.out) + at));
            const uint4 d = __ldg(reinterpret_cast<const uint4*>(
                static_cast<const T*>(g.dout) + b * g.dos[0] + l * g.dos[1] + h * g.dos[2] + 8 * c));
            uint4 r = make_uint4(0, 0, 0, 0);
            if (p.residue)
                r = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.residue) + at));
            const T *op = reinterpret_cast<const T*>(&o), *dp = reinterpret_cast<const T*>(&d),
                    *rp = reinterpret_cast<const T*>(&r);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = to_acc(dp[i]);
                sum += (to_acc(op[i]) + to_acc(rp[i])) * x;
                sq += x * x;
            }
        }
#pragma unroll
        for (int i = LN / 2; i; i >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, i);
            sq += __shfl_xor_sync(0xffffffffu, sq, i);
        }
        if (c == 0 && l < p.Lq) {
            const int64_t at = static_cast<int64_t>(bh) * p.Lq + l;
            if (g.dlse) sum -= static_cast<const float*>(g.dlse)[at];
            const float* stats = static_cast<const float*>(p.stats);
            // (a row that is not finite gives NaN, and does not set the others' scale)
            const float norm = sq < INFINITY ? sqrtf(sq) : 0.f;
            recs[at] = RowRec{stats[at] + (sum - sum), stats[rows + at], sum, norm};
            most = fmaxf(most, norm);
            if (TOPS && fabsf(sum) < INFINITY) most_delta = fmaxf(most_delta, fabsf(sum));
        }
    }
    if (c == 0) {
        top[0][sub] = most;
        if (TOPS) top[1][sub] = most_delta;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < RB; ++i) most = fmaxf(most, top[0][i]);
        norms[blockIdx.x] = most;
        if (TOPS) {
            for (int i = 1; i < RB; ++i) most_delta = fmaxf(most_delta, top[1][i]);
            deltas[blockIdx.x] = most_delta;
        }
    }
}

// The norms of the value rows and the largest of each 128, as above.
template <typename T, int LN>
__global__ __launch_bounds__(256) void value_norm_kernel(Params p, float* norms, float* tops, int blocks_h) {
    constexpr int RB = 256 / LN;
    __shared__ float top[RB];
    const int bh = blockIdx.x / blocks_h, blk = blockIdx.x % blocks_h;
    const int b = bh / p.Hkv, h = bh % p.Hkv, sub = threadIdx.x / LN, c = threadIdx.x % LN;
    const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + h * p.vs[2] + 8 * c;
    float most = 0.f;
#pragma unroll 4
    for (int u = 0; u < kRecRows / RB; ++u) {
        const int l = blk * kRecRows + RB * u + sub;
        float sq = 0.f;
        if (l < p.Lk && 8 * c < p.D) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(v + l * p.vs[1]));
            const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int i = 0; i < 8; ++i) sq += to_acc(x[i]) * to_acc(x[i]);
        }
#pragma unroll
        for (int i = LN / 2; i; i >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, i);
        if (c == 0 && l < p.Lk) {
            const float norm = sq < INFINITY ? sqrtf(sq) : 0.f;
            norms[static_cast<int64_t>(bh) * p.Lk + l] = norm;
            most = fmaxf(most, norm);
        }
    }
    if (c == 0) top[sub] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < RB; ++i) most = fmaxf(most, top[i]);
        tops[blockIdx.x] = most;
    }
}

// The largest norm of the value rows that each query sees, 512 threads a block of 128
// queries.  (In the dq kernel itself, before its first products, it was 8 % of a call.)
__global__ __launch_bounds__(512) void seen_norm_kernel(Params p, const float* norms, const float* tops,
                                                        float* seen, int blocks_h) {
    __shared__ float part_top[4][kRecRows];
    const int bh = blockIdx.x / blocks_h, b = bh / p.Hkv, at = threadIdx.x & 127, part = threadIdx.x >> 7;
    const int row = blockIdx.x % blocks_h * kRecRows + at, n = (p.Lk + kRecRows - 1) / kRecRows;
    const float *one = norms + static_cast<int64_t>(bh) * p.Lk, *block = tops + static_cast<int64_t>(bh) * n;
    int lo = 0, hi = 0;
    if (row < p.Lq) key_span(p, b, row, p.Lk, lo, hi);
    float top = 0.f;
    if (hi > lo)
        over_span(
            lo, hi, p.Lk, part, [&](int i) { top = fmaxf(top, __ldg(one + i)); },
            [&](int i) { top = fmaxf(top, __ldg(block + i)); });
    part_top[part][at] = top;
    __syncthreads();
    if (part || row >= p.Lq) return;
    for (int i = 1; i < 4; ++i) top = fmaxf(top, part_top[i][at]);
    seen[static_cast<int64_t>(bh) * p.Lq + row] = top;
}

bool aligned(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; }

bool boxable(const int64_t* s, int B, int L, int H) {
    const int n[3] = {B, L, H};
    for (int i = 0; i < 3; ++i)
        if (n[i] > 1 && (s[i] <= 0 || s[i] % 8 || s[i] >= (1LL << 38))) return false;
    return true;
}

// Whether the cap's coefficients, up to scale (scale / cap)^10, and the slope's 1 / cap^2 are
// finite in fp32 (infinite ones give NaN where a score is zero).  A cap of a thousandth of
// the scale, or less, takes the kernels that call tanh.
bool cap_in_range(const Params& p) {
    return !(p.cap > 0) || (p.cap > 1e-15 && p.scale * pow(p.scale / p.cap, 10.) < 1e37);
}

}  // namespace

bool encode_heads(CUtensorMap* map, const void* base, const int64_t* strides, int B, int L, int H,
                  int D, bool bf16, const char** err, int rows) {
    auto fn = encoder();
    if (!fn) {
        *err = "cuTensorMapEncodeTiled is unavailable";
        return false;
    }
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(H),
                                static_cast<cuuint64_t>(L), static_cast<cuuint64_t>(B)};
    // the stride of an extent of one is not used, but has to be a valid one
    const cuuint64_t row = 2ull * D;
    const cuuint64_t st[3] = {H > 1 ? 2ull * strides[2] : row, L > 1 ? 2ull * strides[1] : row,
                              B > 1 ? 2ull * strides[0] : row};
    const cuuint32_t box[4] = {64, 1, static_cast<cuuint32_t>(rows), 1}, one[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                    : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                          4, const_cast<void*>(base), dims, st, box, one,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        *err = "cuTensorMapEncodeTiled rejected a layout";
        return false;
    }
    return true;
}

bool tc_fits(const Params& p, int dtype) {
    return (dtype == NSC_F16 || dtype == NSC_BF16) && p.D % 8 == 0 && p.D <= 128 && p.Lk > 0 &&
           !p.lengths && static_cast<float>(p.scale) > 1e-30f && cap_in_range(p) && aligned(p.q) && aligned(p.k) &&
           aligned(p.v) && aligned(p.out) && aligned(p.residue) &&
           boxable(p.qs, p.B, p.Lq, p.Hq) && boxable(p.ks, p.B, p.Lk, p.Hkv) &&
           boxable(p.vs, p.B, p.Lk, p.Hkv);
}

nsc_status tc_fwd(const Params& p, int dtype, cudaStream_t st) {
    if (dtype == NSC_BF16)
        return p.D <= 64 ? tc_fwd_run<__nv_bfloat16, 64>(p, st)
                         : tc_fwd_run<__nv_bfloat16, 128>(p, st);
    return p.D <= 64 ? tc_fwd_run<__half, 64>(p, st) : tc_fwd_run<__half, 128>(p, st);
}

namespace {
int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }
int64_t rec_bytes(int64_t B, int64_t Hq, int64_t Lq) { return round256(B * Hq * Lq * sizeof(RowRec)); }
int64_t rec_blocks(int64_t L) { return (L + kRecRows - 1) / kRecRows; }
int64_t norm_bytes(int64_t B, int64_t Hkv, int64_t L) { return round256(B * Hkv * L * sizeof(float)); }
int64_t top_bytes(int64_t B, int64_t H, int64_t L) { return norm_bytes(B, H, rec_blocks(L)); }
}  // namespace

int64_t tc_bwd_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t Lq, int64_t Lk, int64_t nb) {
    return rec_bytes(B, Hq, Lq) + 2 * top_bytes(B, Hq, Lq) + norm_bytes(B, Hkv, Lk) +
           norm_bytes(B, Hkv, Lq) + top_bytes(B, Hkv, Lk) +
           (nb ? round256(Hq * B * ((Lq + kRows - 1) / kRows) * nb * sizeof(float)) : 0);
}

bool tc_bwd_fits(const Params& p, const Grads& g, int dtype) {
    return tc_fits(p, dtype) && p.Lq > 0 && aligned(g.dout) && aligned(g.dq) && aligned(g.dk) &&
           aligned(g.dv) && boxable(g.dos, p.B, p.Lq, p.Hq);
}

nsc_status tc_bwd(const Params& p, Grads g, void* workspace, void* grad_table, int dtype,
                  cudaStream_t st) {
    char* w = static_cast<char*>(workspace);
    auto take = [&w](int64_t bytes) {
        char* at = w;
        w += bytes;
        return at;
    };
    RowRec* recs = reinterpret_cast<RowRec*>(take(rec_bytes(p.B, p.Hq, p.Lq)));
    float* row_norms = reinterpret_cast<float*>(take(top_bytes(p.B, p.Hq, p.Lq)));
    float *row_deltas = nullptr, *value_norms = nullptr, *seen_norms = nullptr;
    const int n = static_cast<int>(rec_blocks(p.Lq));
    const unsigned blocks = static_cast<unsigned>(p.B) * p.Hq * n;
    if (dtype == NSC_F16) {
        row_deltas = reinterpret_cast<float*>(take(top_bytes(p.B, p.Hq, p.Lq)));
        value_norms = reinterpret_cast<float*>(take(norm_bytes(p.B, p.Hkv, p.Lk)));
        seen_norms = reinterpret_cast<float*>(take(norm_bytes(p.B, p.Hkv, p.Lq)));
        float* tops = reinterpret_cast<float*>(take(top_bytes(p.B, p.Hkv, p.Lk)));
        const int nv = static_cast<int>(rec_blocks(p.Lk));
        auto norms = p.D <= 64 ? value_norm_kernel<__half, 8> : value_norm_kernel<__half, 16>;
        norms<<<static_cast<unsigned>(p.B) * p.Hkv * nv, 256, 0, st>>>(p, value_norms, tops, nv);
        nsc_status r = check_launch("token_attention backward");
        if (r != NSC_OK) return r;
        seen_norm_kernel<<<static_cast<unsigned>(p.B) * p.Hkv * n, 512, 0, st>>>(p, value_norms, tops,
                                                                                seen_norms, n);
        r = check_launch("token_attention backward");
        if (r != NSC_OK) return r;
    }
    g.row_norms = row_norms;
    g.row_deltas = row_deltas;
    g.value_norms = value_norms;
    g.seen_norms = seen_norms;
    if (grad_table) {
        g.tab = w;
        g.n_part = p.B * ((p.Lq + kRows - 1) / kRows);
    }
    auto record = dtype == NSC_BF16 ? (p.D <= 64 ? record_kernel<__nv_bfloat16, 8, false>
                                                 : record_kernel<__nv_bfloat16, 16, false>)
                                    : (p.D <= 64 ? record_kernel<__half, 8, true>
                                                 : record_kernel<__half, 16, true>);
    record<<<blocks, 256, 0, st>>>(p, g, recs, row_norms, row_deltas, n);
    nsc_status r = check_launch("token_attention backward");
    if (r != NSC_OK) return r;
    if (dtype == NSC_BF16)
        r = p.D <= 64 ? tc_bwd_run<__nv_bfloat16, 64>(p, g, recs, st)
                      : tc_bwd_run<__nv_bfloat16, 128>(p, g, recs, st);
    else
        r = p.D <= 64 ? tc_bwd_run<__half, 64>(p, g, recs, st)
                      : tc_bwd_run<__half, 128>(p, g, recs, st);
    if (r == NSC_OK && grad_table) r = launch_table_join(p, g, grad_table, st);
    return r;
}

}  // namespace tok
}  // namespace nsc
