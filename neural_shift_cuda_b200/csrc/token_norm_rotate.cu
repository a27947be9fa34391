// token_norm_rotate.cu -- root-mean-square norm of query and key heads and the
// position rotation, forward and backward, each one pass over the data.
//
//     r = rsqrt(mean(x^2) + eps),  y = x r w,  out = R y
//     h = R^T grad_out,  dw = sum h x r,
//     dx = r h w - x r^3 mean(h w x)
//
// Bound by memory: a head is read once and written once (backward: x and
// grad_out read, dx written).  A group of `LANES` lanes holds one head, 16
// channels a lane as two chunks of 8 half a head apart: both ends of a rotated
// pair are then in the same lane for either pairing, the only exchange is
// that of the sums, and every access is 16 bytes.  A group walks several
// heads of one token with its cosines and sines in registers, the loads of
// up to four heads in flight.
#include "nsc_host.h"

namespace nsc {
namespace rot {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPart = 592;    // blocks that hold weight-gradient partials: 4 an SM

struct Args {
    const void *q, *k, *wq, *wk, *cos, *sin;
    const int32_t* pos;
    int64_t qs[3], ks[3];
    int64_t tokens;       // B * L
    int L, Hq, Hkv, D, R, w_dtype, adjacent, per;   // per: heads of one job
    int64_t rows;
    double eps;
};
struct Out { void *q, *k; };
struct Grad { const void *gq, *gk; void *dq, *dk; void* part; int want_w; };

template <typename A> __device__ __forceinline__ A rsqrt_(A x);
template <> __device__ __forceinline__ float rsqrt_(float x) { return rsqrtf(x); }
template <> __device__ __forceinline__ double rsqrt_(double x) { return 1.0 / sqrt(x); }

template <typename A>
__device__ __forceinline__ A weight_at(const void* w, int dt, int d) {
    if (!w) return A(1);
    switch (dt) {
        case NSC_F16: return to_acc(static_cast<const __half*>(w)[d]);
        case NSC_BF16: return to_acc(static_cast<const __nv_bfloat16*>(w)[d]);
        case NSC_F32: return static_cast<const float*>(w)[d];
    }
    return static_cast<A>(static_cast<const double*>(w)[d]);
}

// 8 values, 16-byte aligned, as raw words
template <typename T> struct Raw { uint4 u[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ Raw<T> load8(const T* p) {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
        r.u[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    return r;
}
template <typename T, typename A>
__device__ __forceinline__ void unpack(const Raw<T>& r, A (&v)[8]) {
    const T* t = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_acc(t[i]);
}
template <typename T> __device__ __forceinline__ T cast_to(float v) { return from_float<T>(v); }
template <typename T> __device__ __forceinline__ T cast_to(double v) { return v; }
template <typename T, typename A>
__device__ __forceinline__ void store8(T* p, const A (&v)[8]) {
    Raw<T> r;
    T* t = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = cast_to<T>(v[i]);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
        reinterpret_cast<uint4*>(p)[i] = r.u[i];
}

// Cosines and sines of a lane's 8 pairs at a position; outside the table NaN.
template <typename A>
__device__ __forceinline__ void turn_at(const Args& a, int64_t pos, int c, int adjacent, A (&cs)[8],
                                        A (&sn)[8]) {
    const bool in = pos >= 0 && pos < a.rows;
    const A* cp = static_cast<const A*>(a.cos) + (in ? pos : 0) * (a.D / 2);
    const A* sp = static_cast<const A*>(a.sin) + (in ? pos : 0) * (a.D / 2);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int at = adjacent ? (i < 4 ? 4 * c + i : a.D / 4 + 4 * c + i - 4) : 8 * c + i;
        cs[i] = in ? __ldg(cp + at) : static_cast<A>(NAN);
        sn[i] = in ? __ldg(sp + at) : static_cast<A>(NAN);
    }
}

// Turns the lane's pairs in place; back: by the opposite angle.
template <typename A, bool ADJ, bool BACK>
__device__ __forceinline__ void turn(A (&x)[8], A (&y)[8], const A (&cs)[8], const A (&sn)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        A& u = ADJ ? (i < 4 ? x[2 * (i & 3)] : y[2 * (i & 3)]) : x[i];
        A& v = ADJ ? (i < 4 ? x[2 * (i & 3) + 1] : y[2 * (i & 3) + 1]) : y[i];
        const A s = BACK ? -sn[i] : sn[i];
        const A a = u * cs[i] - v * s, b = v * cs[i] + u * s;
        u = a;
        v = b;
    }
}

template <typename A, int LANES>
__device__ __forceinline__ A group_sum(A v) {
#pragma unroll
    for (int i = 1; i < LANES; i <<= 1) v += __shfl_xor_sync(0xffffffffu, v, i);
    return v;
}

// A job is `per` heads of q, or of k, of one token.
struct Job { int64_t token; bool is_k; int h0, h1; };
__device__ __forceinline__ Job job_at(const Args& a, int64_t j, int nq, int nk) {
    Job r;
    r.token = j / (nq + nk);
    const int c = static_cast<int>(j - r.token * (nq + nk));
    r.is_k = c >= nq;
    r.h0 = (r.is_k ? c - nq : c) * a.per;
    r.h1 = min(r.h0 + a.per, r.is_k ? a.Hkv : a.Hq);
    return r;
}

template <typename T, typename A, int LANES, bool ADJ>
__global__ __launch_bounds__(kThreads) void fwd_kernel(Args a, Out o, int nq, int nk) {
    constexpr int U = sizeof(T) == 2 ? 4 : 2;   // heads in flight
    const int c = threadIdx.x % LANES, half = a.D / 2;
    const int64_t j = static_cast<int64_t>(blockIdx.x) * (kThreads / LANES) + threadIdx.x / LANES;
    const bool work = j < a.tokens * (nq + nk), lane_on = work && 8 * c < half;
    Job jb = job_at(a, work ? j : 0, nq, nk);
    const int64_t b = jb.token / a.L, l = jb.token - b * a.L;
    const int H = jb.is_k ? a.Hkv : a.Hq;
    const int64_t* st = jb.is_k ? a.ks : a.qs;
    const T* src = static_cast<const T*>(jb.is_k ? a.k : a.q) + b * st[0] + l * st[1] + 8 * c;
    T* dst = static_cast<T*>(jb.is_k ? o.k : o.q) + jb.token * H * a.D + 8 * c;
    A cs[8], sn[8], w[16];
    if (lane_on) {
        turn_at<A>(a, a.pos ? __ldg(a.pos + jb.token) : l, c, ADJ, cs, sn);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            w[i] = weight_at<A>(jb.is_k ? a.wk : a.wq, a.w_dtype,
                                (i < 8 ? 0 : half - 8) + 8 * c + i);
    }
    // all lanes of a warp take part in the exchanges: the trip count is `per`
    for (int h0 = jb.h0; h0 < jb.h0 + a.per; h0 += U) {
        Raw<T> rx[U], ry[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (lane_on && h0 + u < jb.h1) {
                rx[u] = load8<T>(src + (h0 + u) * st[2]);
                ry[u] = load8<T>(src + (h0 + u) * st[2] + half);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool on = lane_on && h0 + u < jb.h1;
            A x[8], y[8], sq = 0;
            if (on) {
                unpack<T>(rx[u], x);
                unpack<T>(ry[u], y);
#pragma unroll
                for (int i = 0; i < 8; ++i) sq += x[i] * x[i] + y[i] * y[i];
            }
            sq = group_sum<A, LANES>(sq);
            if (!on) continue;
            const A r = rsqrt_<A>(sq / a.D + static_cast<A>(a.eps));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] *= r * w[i];
                y[i] *= r * w[8 + i];
            }
            turn<A, ADJ, false>(x, y, cs, sn);
            T* d = dst + static_cast<int64_t>(h0 + u) * a.D;
            store8<T>(d, x);
            store8<T>(d + half, y);
        }
    }
}

// Blocks [0, q_blocks) pass over q, the others over k, so that a thread holds the
// weight sums of one of them.
template <typename T, typename A, int LANES, bool ADJ>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void bwd_kernel(Args a, Grad g,
                                                                              int q_blocks) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    constexpr int GROUPS = kThreads / LANES;
    constexpr int U = 2;
    const int c = threadIdx.x % LANES, half = a.D / 2;
    const bool is_k = static_cast<int>(blockIdx.x) >= q_blocks, lane_in = 8 * c < half;
    const int H = is_k ? a.Hkv : a.Hq, chunks = (H + a.per - 1) / a.per;
    const int64_t s0 = is_k ? a.ks[0] : a.qs[0], s1 = is_k ? a.ks[1] : a.qs[1];
    const int64_t s2 = is_k ? a.ks[2] : a.qs[2];
    const T* src = static_cast<const T*>(is_k ? a.k : a.q) + 8 * c;
    const T* gsrc = static_cast<const T*>(is_k ? g.gk : g.gq) + 8 * c;
    T* dst = static_cast<T*>(is_k ? g.dk : g.dq) + 8 * c;
    A dw[16], w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        dw[i] = 0;
        w[i] = lane_in ? weight_at<A>(is_k ? a.wk : a.wq, a.w_dtype, (i < 8 ? 0 : half - 8) + 8 * c + i)
                       : A(0);
    }
    const int first = is_k ? static_cast<int>(blockIdx.x) - q_blocks : static_cast<int>(blockIdx.x);
    const int blocks = is_k ? static_cast<int>(gridDim.x) - q_blocks : q_blocks;
    const int64_t jobs = a.tokens * chunks, step = static_cast<int64_t>(blocks) * GROUPS;
    const A inv_d = A(1) / a.D;
    // all lanes of the block make the same number of rounds
    for (int64_t j0 = static_cast<int64_t>(first) * GROUPS; j0 < jobs; j0 += step) {
        const int64_t j = j0 + threadIdx.x / LANES;
        const bool lane_on = j < jobs && lane_in;
        const int64_t token = j < jobs ? j / chunks : 0;
        const int h_first = j < jobs ? static_cast<int>(j - token * chunks) * a.per : 0;
        const int h_end = min(h_first + a.per, H);
        const int64_t b = token / a.L, l = token - b * a.L;
        const T* x_at = src + b * s0 + l * s1;
        const int64_t row0 = token * H;
        A cs[8], sn[8];
        if (lane_on) turn_at<A>(a, a.pos ? __ldg(a.pos + token) : l, c, ADJ, cs, sn);
        for (int h0 = h_first; h0 < h_first + a.per; h0 += U) {
            Raw<T> rx[U], ry[U], rg[U], ri[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (lane_on && h0 + u < h_end) {
                    rx[u] = load8<T>(x_at + (h0 + u) * s2);
                    ry[u] = load8<T>(x_at + (h0 + u) * s2 + half);
                    rg[u] = load8<T>(gsrc + (row0 + h0 + u) * a.D);
                    ri[u] = load8<T>(gsrc + (row0 + h0 + u) * a.D + half);
                }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool on = lane_on && h0 + u < h_end;
                A x[8], y[8], p[8], q[8], sq = 0, dot = 0;
                if (on) {
                    unpack<T>(rx[u], x);
                    unpack<T>(ry[u], y);
                    unpack<T>(rg[u], p);
                    unpack<T>(ri[u], q);
                    turn<A, ADJ, true>(p, q, cs, sn);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        sq += x[i] * x[i] + y[i] * y[i];
                        dot += p[i] * w[i] * x[i] + q[i] * w[8 + i] * y[i];
                    }
                }
                sq = group_sum<A, LANES>(sq);
                dot = group_sum<A, LANES>(dot);
                if (!on) continue;
                const A r = rsqrt_<A>(sq * inv_d + static_cast<A>(a.eps));
                const A f = r * r * r * dot * inv_d;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    p[i] *= r;
                    q[i] *= r;
                    dw[i] += p[i] * x[i];
                    dw[8 + i] += q[i] * y[i];
                    x[i] = p[i] * w[i] - x[i] * f;
                    y[i] = q[i] * w[8 + i] - y[i] * f;
                }
                T* d = dst + (row0 + h0 + u) * a.D;
                store8<T>(d, x);
                store8<T>(d + half, y);
            }
        }
    }
    if (!g.want_w) return;
    // groups of a warp, then the warps, in a fixed order
    A* sh = reinterpret_cast<A*>(smem_raw);   // [warps][16 * LANES]
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        A v = dw[i];
#pragma unroll
        for (int m = LANES; m < 32; m <<= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
        if (lane < LANES) sh[warp * 16 * LANES + (i < 8 ? 0 : 8 * LANES) + 8 * c + (i & 7)] = v;
    }
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += kThreads) {
        const int at = d < half ? d : 8 * LANES + d - half;
        A v = 0;
        for (int k = 0; k < kThreads / 32; ++k) v += sh[k * 16 * LANES + at];
        static_cast<A*>(g.part)[static_cast<int64_t>(blockIdx.x) * a.D + d] = v;
    }
}

// Any D, R, stride and alignment: a warp a head, channels a lane apart.
template <typename T, typename A>
__global__ __launch_bounds__(kThreads) void any_kernel(Args a, Out o, Grad g, int back) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = kThreads / 32;
    A* h = reinterpret_cast<A*>(smem_raw) + warp * a.D;                  // turned-back gradient
    A* dw = reinterpret_cast<A*>(smem_raw) + warps * a.D + warp * 2 * a.D;
    if (back)
        for (int d = lane; d < 2 * a.D; d += 32) dw[d] = 0;
    const int heads = a.Hq + a.Hkv;
    const int64_t jobs = a.tokens * heads, step = static_cast<int64_t>(gridDim.x) * warps;
    for (int64_t j = static_cast<int64_t>(blockIdx.x) * warps + warp; j < jobs; j += step) {
        const int64_t token = j / heads, b = token / a.L, l = token - b * a.L;
        int hd = static_cast<int>(j - token * heads);
        const bool is_k = hd >= a.Hq;
        if (is_k) hd -= a.Hq;
        const int H = is_k ? a.Hkv : a.Hq;
        const int64_t* st = is_k ? a.ks : a.qs;
        const void* w = is_k ? a.wk : a.wq;
        const T* x = static_cast<const T*>(is_k ? a.k : a.q) + b * st[0] + l * st[1] + hd * st[2];
        const int64_t at = (token * H + hd) * a.D, pos = a.pos ? a.pos[token] : l;
        const bool in = pos >= 0 && pos < a.rows;
        const A* cp = static_cast<const A*>(a.cos) + (in ? pos : 0) * (a.R / 2);
        const A* sp = static_cast<const A*>(a.sin) + (in ? pos : 0) * (a.R / 2);
        A sq = 0;
        for (int d = lane; d < a.D; d += 32) sq += static_cast<A>(to_acc(x[d])) * static_cast<A>(to_acc(x[d]));
        sq = group_sum<A, 32>(sq);
        const A r = rsqrt_<A>(sq / a.D + static_cast<A>(a.eps));
        // pair i: channels u, v; past the turned ones a pair is two channels
        if (!back) {
            T* d = static_cast<T*>(is_k ? o.k : o.q) + at;
            for (int i = lane; i < a.D / 2; i += 32) {
                const bool t = i < a.R / 2;
                const int u = t && !a.adjacent ? i : 2 * i, v = t && !a.adjacent ? i + a.R / 2 : u + 1;
                const A p = static_cast<A>(to_acc(x[u])) * r * weight_at<A>(w, a.w_dtype, u);
                const A q = static_cast<A>(to_acc(x[v])) * r * weight_at<A>(w, a.w_dtype, v);
                const A cs = !t ? A(1) : in ? cp[i] : static_cast<A>(NAN);
                const A sn = !t ? A(0) : in ? sp[i] : static_cast<A>(NAN);
                d[u] = cast_to<T>(t ? p * cs - q * sn : p);
                d[v] = cast_to<T>(t ? q * cs + p * sn : q);
            }
            continue;
        }
        const T* go = static_cast<const T*>(is_k ? g.gk : g.gq) + at;
        T* d = static_cast<T*>(is_k ? g.dk : g.dq) + at;
        A dot = 0;
        for (int i = lane; i < a.D / 2; i += 32) {
            const bool t = i < a.R / 2;
            const int u = t && !a.adjacent ? i : 2 * i, v = t && !a.adjacent ? i + a.R / 2 : u + 1;
            const A p = to_acc(go[u]), q = to_acc(go[v]);
            const A cs = !t ? A(1) : in ? cp[i] : static_cast<A>(NAN);
            const A sn = !t ? A(0) : in ? sp[i] : static_cast<A>(NAN);
            h[u] = t ? p * cs + q * sn : p;
            h[v] = t ? q * cs - p * sn : q;
        }
        __syncwarp();
        for (int i = lane; i < a.D; i += 32)
            dot += h[i] * weight_at<A>(w, a.w_dtype, i) * static_cast<A>(to_acc(x[i]));
        dot = group_sum<A, 32>(dot);
        const A f = r * r * r * dot / a.D;
        for (int i = lane; i < a.D; i += 32) {
            const A xi = to_acc(x[i]);
            dw[(is_k ? a.D : 0) + i] += h[i] * xi * r;
            d[i] = cast_to<T>(r * h[i] * weight_at<A>(w, a.w_dtype, i) - xi * f);
        }
        __syncwarp();
    }
    if (!back || !g.want_w) return;
    __syncthreads();
    const A* all = reinterpret_cast<A*>(smem_raw) + warps * a.D;
    // (a block has a row of sums of q, and further on one of k)
    for (int i = threadIdx.x; i < 2 * a.D; i += kThreads) {
        A v = 0;
        for (int k = 0; k < warps; ++k) v += all[k * 2 * a.D + i];
        const int64_t row = blockIdx.x + (i < a.D ? 0 : gridDim.x);
        static_cast<A*>(g.part)[row * a.D + (i < a.D ? i : i - a.D)] = v;
    }
}

// Sums of the blocks' partials, rows [0, nq) of q and [nq, n) of k: a block 32 columns
// of one of them, its 32 warps side by side over the rows.
template <typename A>
__global__ __launch_bounds__(1024) void join_kernel(const A* part, int nq, int n, int D, void* wq,
                                                    void* wk, int dt) {
    __shared__ A sh[32][33];
    const bool is_k = blockIdx.y == 1;
    void* w = is_k ? wk : wq;
    if (!w) return;
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, d = blockIdx.x * 32 + x;
    const int r0 = is_k ? nq : 0, r1 = is_k ? n : nq;
    A v = 0;
    if (d < D)
#pragma unroll 8
        for (int r = r0 + y; r < r1; r += 32) v += part[static_cast<int64_t>(r) * D + d];
    sh[y][x] = v;
    __syncthreads();
    // warp y sums column y
    v = sh[x][y];
#pragma unroll
    for (int i = 16; i; i >>= 1) v += __shfl_xor_sync(0xffffffffu, v, i);
    const int o = blockIdx.x * 32 + y;
    if (x || o >= D) return;
    switch (dt) {
        case NSC_F16: static_cast<__half*>(w)[o] = __float2half_rn(static_cast<float>(v)); break;
        case NSC_BF16:
            static_cast<__nv_bfloat16*>(w)[o] = __float2bfloat16_rn(static_cast<float>(v));
            break;
        case NSC_F32: static_cast<float*>(w)[o] = static_cast<float>(v); break;
        default: static_cast<double*>(w)[o] = v;
    }
}

nsc_status check(const char* op, const nsc_norm_rotate* a) {
    if (!a) return fail(NSC_ERR_INVALID_ARG, "%s: arguments are NULL", op);
    if (!valid_dtype(a->dtype))
        return fail(NSC_ERR_UNSUPPORTED_DTYPE, "%s: unsupported dtype code %d", op, a->dtype);
    if (a->B < 0 || a->L < 0 || a->Hq < 0 || a->Hkv < 0 || a->rows < 0)
        return fail(NSC_ERR_INVALID_ARG, "%s: bad extent", op);
    if (a->D < 2 || a->D > 512 || a->D % 2)
        return fail(NSC_ERR_INVALID_ARG, "%s: head width %lld is not even and in 2..512", op,
                    (long long)a->D);
    if (a->rot_dim < 0 || a->rot_dim > a->D || a->rot_dim % 2)
        return fail(NSC_ERR_INVALID_ARG, "%s: %lld turned channels of %lld", op,
                    (long long)a->rot_dim, (long long)a->D);
    if (a->L >= (1LL << 31) || a->Hq >= (1LL << 20) || a->Hkv >= (1LL << 20) ||
        (a->L && a->B >= (1LL << 31) / a->L))
        return fail(NSC_ERR_INVALID_ARG, "%s: too many tokens", op);
    const bool half = a->dtype == NSC_F16 || a->dtype == NSC_BF16;
    if ((a->q_weight || a->k_weight) && a->weight_dtype != a->dtype &&
        !(half && a->weight_dtype == NSC_F32))
        return fail(NSC_ERR_UNSUPPORTED_DTYPE,
                    "%s: a weight has the dtype of q, or fp32 with fp16 / bf16", op);
    if (!(a->eps >= 0)) return fail(NSC_ERR_INVALID_ARG, "%s: eps must be >= 0", op);
    const bool any = a->B && a->L;
    if ((any && a->Hq && !a->q) || (any && a->Hkv && !a->k) ||
        (any && a->rot_dim && a->rows && (!a->cos || !a->sin)))
        return fail(NSC_ERR_INVALID_ARG, "%s: NULL pointer", op);
    return ok();
}

Args args(const nsc_norm_rotate* a) {
    Args r{};
    r.q = a->q; r.k = a->k; r.wq = a->q_weight; r.wk = a->k_weight;
    r.cos = a->cos; r.sin = a->sin; r.pos = a->positions;
    for (int i = 0; i < 3; ++i) { r.qs[i] = a->q_stride[i]; r.ks[i] = a->k_stride[i]; }
    r.tokens = a->B * a->L;
    r.L = static_cast<int>(a->L);
    r.Hq = static_cast<int>(a->Hq);
    r.Hkv = static_cast<int>(a->Hkv);
    r.D = static_cast<int>(a->D);
    r.R = static_cast<int>(a->rot_dim);
    r.rows = a->rows;
    r.w_dtype = a->weight_dtype;
    r.adjacent = a->adjacent != 0;
    r.eps = a->eps;
    return r;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether 16-byte accesses of whole chunks serve this call.
bool wide(const nsc_norm_rotate* a) {
    const int64_t es = dtype_size(a->dtype);
    // (fp64 would spill its two chunks; it takes the other kernel)
    bool w = a->dtype != NSC_F64 && a->D % 16 == 0 && a->rot_dim == a->D && a->rows > 0 && aligned16(a->q) &&
             aligned16(a->k);
    for (int i = 0; i < 3; ++i)
        w = w && a->q_stride[i] * es % 16 == 0 && a->k_stride[i] * es % 16 == 0;
    return w;
}

int lanes_for(int D) {
    int n = 1;
    while (n * 16 < D) n <<= 1;
    return n;
}

// Heads of one job: all of a token's share its cosines and sines, but a call
// of few tokens is spread over more groups.
int heads_per_job(const Args& a, int lanes) {
    const int most = a.Hq > a.Hkv ? a.Hq : a.Hkv;
    int per = 1;
    while (per < 8 && per < most &&
           a.tokens * ((a.Hq + 2 * per - 1) / (2 * per) + (a.Hkv + 2 * per - 1) / (2 * per)) *
                   lanes >= 148LL * 1024)
        per <<= 1;
    return per;
}

template <typename T, typename A, int LANES>
nsc_status run_wide(Args a, const Out* o, const Grad* g, int* n_part, cudaStream_t st) {
    a.per = heads_per_job(a, LANES);
    const int nq = (a.Hq + a.per - 1) / a.per, nk = (a.Hkv + a.per - 1) / a.per;
    const int64_t jobs = a.tokens * (nq + nk);
    const int64_t blocks = (jobs + kThreads / LANES - 1) / (kThreads / LANES);
    if (o) {
        if (blocks >= (1LL << 31)) return fail(NSC_ERR_INVALID_ARG, "qk_norm_rotate: too many tokens");
        const unsigned n = static_cast<unsigned>(blocks);
        if (a.adjacent) fwd_kernel<T, A, LANES, true><<<n, kThreads, 0, st>>>(a, *o, nq, nk);
        else fwd_kernel<T, A, LANES, false><<<n, kThreads, 0, st>>>(a, *o, nq, nk);
        return check_launch("qk_norm_rotate");
    }
    // blocks of q and of k in the ratio of their work, two rounds an SM at most
    constexpr int groups = kThreads / LANES;
    int64_t bq = (a.tokens * nq + groups - 1) / groups, bk = (a.tokens * nk + groups - 1) / groups;
    if (bq + bk > kMaxPart) {
        const int64_t all = static_cast<int64_t>(a.Hq) + a.Hkv;
        bk = a.Hkv ? (kMaxPart * static_cast<int64_t>(a.Hkv) + all - 1) / all : 0;
        bq = kMaxPart - bk;
        if (a.Hq && bq < 1) { bq = 1; bk = kMaxPart - 1; }
    }
    n_part[0] = static_cast<int>(bq);
    n_part[1] = static_cast<int>(bq + bk);
    const size_t smem = sizeof(A) * (kThreads / 32) * 16 * LANES;
    auto kern = a.adjacent ? bwd_kernel<T, A, LANES, true> : bwd_kernel<T, A, LANES, false>;
    kern<<<n_part[1], kThreads, smem, st>>>(a, *g, n_part[0]);
    return check_launch("qk_norm_rotate backward");
}

template <typename T, typename A>
nsc_status run(const nsc_norm_rotate* n, const Out* o, const Grad* g, int* n_part,
               cudaStream_t st) {
    Args a = args(n);
    if constexpr (sizeof(T) < 8) if (wide(n)) {
        switch (lanes_for(a.D)) {
            case 1: return run_wide<T, A, 1>(a, o, g, n_part, st);
            case 2: return run_wide<T, A, 2>(a, o, g, n_part, st);
            case 4: return run_wide<T, A, 4>(a, o, g, n_part, st);
            case 8: return run_wide<T, A, 8>(a, o, g, n_part, st);
            case 16: return run_wide<T, A, 16>(a, o, g, n_part, st);
            default: return run_wide<T, A, 32>(a, o, g, n_part, st);
        }
    }
    const int warps = kThreads / 32;
    int64_t blocks = (a.tokens * (a.Hq + a.Hkv) + warps - 1) / warps;
    if (blocks > kMaxPart) blocks = kMaxPart;
    if (n_part) {
        n_part[0] = static_cast<int>(blocks);
        n_part[1] = static_cast<int>(2 * blocks);
    }
    const size_t smem = g ? sizeof(A) * warps * 3 * a.D : 0;
    if (smem > 48 * 1024)
        cudaFuncSetAttribute(any_kernel<T, A>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(smem));
    any_kernel<T, A><<<static_cast<unsigned>(blocks), kThreads, smem, st>>>(
        a, o ? *o : Out{}, g ? *g : Grad{}, g ? 1 : 0);
    return check_launch("qk_norm_rotate");
}

nsc_status dispatch(const nsc_norm_rotate* n, const Out* o, const Grad* g, int* n_part,
                    cudaStream_t st) {
    switch (n->dtype) {
        case NSC_F16: return run<__half, float>(n, o, g, n_part, st);
        case NSC_BF16: return run<__nv_bfloat16, float>(n, o, g, n_part, st);
        case NSC_F32: return run<float, float>(n, o, g, n_part, st);
        default: return run<double, double>(n, o, g, n_part, st);
    }
}

}  // namespace
}  // namespace rot
}  // namespace nsc

using namespace nsc;
using namespace nsc::rot;

extern "C" NSC_API nsc_status nsc_qk_norm_rotate_fwd(const nsc_norm_rotate* a, void* q_out,
                                                     void* k_out, void* stream) {
    const char* op = "qk_norm_rotate";
    nsc_status st = rot::check(op, a);
    if (st != NSC_OK) return st;
    if (!a->B || !a->L || !(a->Hq + a->Hkv)) return ok();
    if ((a->Hq && !q_out) || (a->Hkv && !k_out))
        return fail(NSC_ERR_INVALID_ARG, "%s: NULL pointer", op);
    const Out o{q_out, k_out};
    return dispatch(a, &o, nullptr, nullptr, as_stream(stream));
}

extern "C" NSC_API int64_t nsc_qk_norm_rotate_workspace(const nsc_norm_rotate* a) {
    if (rot::check("qk_norm_rotate", a) != NSC_OK) return -1;
    return static_cast<int64_t>(kMaxPart) * 2 * a->D * (a->dtype == NSC_F64 ? 8 : 4);
}

extern "C" NSC_API nsc_status nsc_qk_norm_rotate_bwd(const nsc_norm_rotate* a,
                                                     const void* grad_q_out,
                                                     const void* grad_k_out, void* grad_q,
                                                     void* grad_k, void* grad_q_weight,
                                                     void* grad_k_weight, void* workspace,
                                                     void* stream) {
    const char* op = "qk_norm_rotate backward";
    nsc_status st = rot::check(op, a);
    if (st != NSC_OK) return st;
    const bool want = grad_q_weight || grad_k_weight, any = a->B && a->L;
    if ((any && a->Hq && (!grad_q_out || !grad_q)) || (any && a->Hkv && (!grad_k_out || !grad_k)) ||
        (want && !workspace) || (grad_q_weight && !a->q_weight) || (grad_k_weight && !a->k_weight))
        return fail(NSC_ERR_INVALID_ARG, "%s: NULL pointer", op);
    cudaStream_t s = as_stream(stream);
    int n_part[2] = {0, 0};
    if (any && a->Hq + a->Hkv) {
        const Grad g{grad_q_out, grad_k_out, grad_q, grad_k, workspace, want};
        st = dispatch(a, nullptr, &g, n_part, s);
        if (st != NSC_OK) return st;
    }
    if (!want) return ok();
    const dim3 blocks(static_cast<unsigned>((a->D + 31) / 32), 2);
    if (a->dtype == NSC_F64)
        join_kernel<double><<<blocks, 1024, 0, s>>>(static_cast<const double*>(workspace), n_part[0],
                                                    n_part[1], static_cast<int>(a->D),
                                                    grad_q_weight, grad_k_weight, a->weight_dtype);
    else
        join_kernel<float><<<blocks, 1024, 0, s>>>(static_cast<const float*>(workspace), n_part[0],
                                                   n_part[1], static_cast<int>(a->D),
                                                   grad_q_weight, grad_k_weight, a->weight_dtype);
    return check_launch(op);
}
