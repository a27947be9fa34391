// token_norm_rotate.cu -- root-mean-square norm of query and key heads and the
// position rotation, forward and backward, each one pass over the data.
//
//     r = rsqrt(mean(x^2) + eps),  y = x r w,  out = R y
//     h = R^T grad_out,  dw = sum h x r,
//     dx = r h w - x r^3 mean(h w x)
//
// Bound by memory: a head is read once and written once (backward: x and
// grad_out read, dx written).  A group of `LANES` lanes holds one head, 8
// channels a lane as two chunks of 4 half a head apart (past 256 channels, two of 8):
// both ends of a rotated pair are then in the same lane for either pairing, and the
// only exchange is that of the sums.  A group walks the heads of a token with its
// cosines and sines in registers; as soon as a head is unpacked, the load of the one
// four further on takes its place, across tokens too.  Arithmetic is two pairs an
// instruction: at one each it took as long as the memory.
//
// 4 x 4096 tokens, 16 + 16 heads of 128, bf16 (slices of a projection): forward 49 us for
// 268 MB (5.4 TB/s of the 6.5 that a copy reaches), backward 79 us for 403 MB (5.1
// TB/s).  Before: blocks of one round each, 16 channels a lane, one pair an instruction:
// 62 and 104 us.
#include <type_traits>

#include "nsc_host.h"

namespace nsc {
namespace rot {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPart = 592;   // most rows of weight-gradient partials of a tensor
// Resident blocks an SM, by registers (forward: with 4 of 64 registers 52 us, with 2 55 us;
// backward: with 3 of 80 it spills, 134 us).
constexpr int kFwdPerSm = 3, kBwdPerSm = 2;
constexpr int kAhead = 4;   // heads in flight a group (16-bit types)

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

// V values as raw words, read in accesses of up to 16 bytes
template <typename T, int V> struct Raw {
    static constexpr int kBytes = V * sizeof(T), kWord = kBytes < 16 ? kBytes : 16;
    using Word = typename std::conditional<kWord == 16, uint4, uint2>::type;
    Word u[kBytes / kWord];
};
template <int V, typename T>
__device__ __forceinline__ Raw<T, V> load(const T* p) {
    using R = Raw<T, V>;
    R r;
#pragma unroll
    for (int i = 0; i < R::kBytes / R::kWord; ++i)
        r.u[i] = __ldg(reinterpret_cast<const typename R::Word*>(p) + i);
    return r;
}
template <typename T> __device__ __forceinline__ T cast_to(float v) { return from_float<T>(v); }
template <typename T> __device__ __forceinline__ T cast_to(double v) { return v; }

// A lane's V pairs (u, v), two by two: channels x of the first half of the head and y of
// the second are u and v (ADJ: neighbours in x, then neighbours in y).
template <int V> struct Pairs { float2 u[V / 2], v[V / 2]; };
template <int V, bool ADJ>
__device__ __forceinline__ Pairs<V> pairs_of(const float (&x)[V], const float (&y)[V]) {
    Pairs<V> p;
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
        if (ADJ) {
            const float(&t)[V] = i < V / 4 ? x : y;
            const int e = 4 * (i % (V / 4));
            p.u[i] = make_float2(t[e], t[e + 2]);
            p.v[i] = make_float2(t[e + 1], t[e + 3]);
        } else {
            p.u[i] = make_float2(x[2 * i], x[2 * i + 1]);
            p.v[i] = make_float2(y[2 * i], y[2 * i + 1]);
        }
    return p;
}
template <bool ADJ, typename T, int V>
__device__ __forceinline__ Pairs<V> unpack(const Raw<T, V>& rx, const Raw<T, V>& ry) {
    float x[V], y[V];
    const T *tx = reinterpret_cast<const T*>(&rx), *ty = reinterpret_cast<const T*>(&ry);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        x[i] = to_acc(tx[i]);
        y[i] = to_acc(ty[i]);
    }
    return pairs_of<V, ADJ>(x, y);
}
template <bool ADJ, typename T, int V>
__device__ __forceinline__ void store(T* d, int half, const Pairs<V>& p) {
    using R = Raw<T, V>;
    R rx, ry;
    T *tx = reinterpret_cast<T*>(&rx), *ty = reinterpret_cast<T*>(&ry);
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
        if (ADJ) {
            T* t = i < V / 4 ? tx : ty;
            const int e = 4 * (i % (V / 4));
            t[e] = cast_to<T>(p.u[i].x);
            t[e + 1] = cast_to<T>(p.v[i].x);
            t[e + 2] = cast_to<T>(p.u[i].y);
            t[e + 3] = cast_to<T>(p.v[i].y);
        } else {
            tx[2 * i] = cast_to<T>(p.u[i].x);
            tx[2 * i + 1] = cast_to<T>(p.u[i].y);
            ty[2 * i] = cast_to<T>(p.v[i].x);
            ty[2 * i + 1] = cast_to<T>(p.v[i].y);
        }
#pragma unroll
    for (int i = 0; i < R::kBytes / R::kWord; ++i) {
        reinterpret_cast<typename R::Word*>(d)[i] = rx.u[i];
        reinterpret_cast<typename R::Word*>(d + half)[i] = ry.u[i];
    }
}

__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 neg(float2 v) { return make_float2(-v.x, -v.y); }

// Cosines and sines of a lane's pairs at a position; outside the table NaN.
template <int V> struct Angles { float2 c[V / 2], s[V / 2]; };
template <int V, bool ADJ>
__device__ __forceinline__ Angles<V> angles_at(const Args& a, int64_t pos, int c) {
    const bool in = pos >= 0 && pos < a.rows;
    const int64_t row = (in ? pos : 0) * (a.D / 2);
    const float *cp = static_cast<const float*>(a.cos) + row, *sp = static_cast<const float*>(a.sin) + row;
    Angles<V> r;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        const int at = ADJ ? (i < V / 4 ? 0 : a.D / 4 - V / 2) + V / 2 * c + 2 * i : V * c + 2 * i;
        r.c[i] = in ? make_float2(__ldg(cp + at), __ldg(cp + at + 1)) : twice(NAN);
        r.s[i] = in ? make_float2(__ldg(sp + at), __ldg(sp + at + 1)) : twice(NAN);
    }
    return r;
}

// Sums over a head's lanes, of N values side by side.
template <int LANES, int N>
__device__ __forceinline__ void group_sums(float (&v)[N]) {
#pragma unroll
    for (int i = 1; i < LANES; i <<= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], i);
}
template <typename A, int LANES>
__device__ __forceinline__ A group_sum(A v) {
#pragma unroll
    for (int i = 1; i < LANES; i <<= 1) v += __shfl_xor_sync(0xffffffffu, v, i);
    return v;
}

// A block's share of the work: blocks [0, q_blocks) pass over q, the others over k, so
// that a thread has one tensor's weights (and weight sums).  A job is `per` heads of one
// token; a group takes every `step`-th job.
template <typename T> struct Share {
    bool is_k;
    int H, chunks, per, L;
    int64_t s0, s1, s2, jobs, first, step;
    const T* src;

    __device__ __forceinline__ Share(const Args& a, int q_blocks, int groups) {
        const int block = static_cast<int>(blockIdx.x);
        is_k = block >= q_blocks;
        H = is_k ? a.Hkv : a.Hq;
        per = a.per;
        L = a.L;
        chunks = (H + per - 1) / per;
        s0 = is_k ? a.ks[0] : a.qs[0];
        s1 = is_k ? a.ks[1] : a.qs[1];
        s2 = is_k ? a.ks[2] : a.qs[2];
        jobs = a.tokens * chunks;
        first = static_cast<int64_t>(is_k ? block - q_blocks : block) * groups;
        step = static_cast<int64_t>(is_k ? static_cast<int>(gridDim.x) - q_blocks : q_blocks) * groups;
        src = static_cast<const T*>(is_k ? a.k : a.q);
    }
};
// Heads [h, end) of a token: x in place, the contiguous tensors at row token H + h.
// Where there is no such head (past a job, past the jobs) reads take the job's first one
// or that of token 0, so that no load waits for a branch; nothing is written then.
template <typename T> struct Spot {
    const T* x;
    int64_t row, token;
    int left;   // heads from here on

    __device__ __forceinline__ Spot(const Share<T>& s, int64_t j) {
        const bool on = j < s.jobs;
        token = on ? static_cast<int64_t>(static_cast<uint64_t>(j) / static_cast<unsigned>(s.chunks)) : 0;
        const int h = on ? static_cast<int>(j - token * s.chunks) * s.per : 0;
        left = on ? min(s.per, s.H - h) : 0;
        const int64_t b = token / s.L;
        x = s.src + b * s.s0 + (token - b * s.L) * s.s1 + h * s.s2;
        row = token * s.H + h;
    }
    __device__ __forceinline__ Spot after(const Share<T>& s, int n) const {
        Spot r = *this;
        r.left = left - n;
        if (r.left > 0) {
            r.x += n * s.s2;
            r.row += n;
        }
        return r;
    }
};
__device__ __forceinline__ int64_t position(const Args& a, int64_t token) {
    return a.pos ? __ldg(a.pos + token) : token % a.L;
}

// Weights of a lane's pairs, kept as fp32 in shared memory.
template <int V, bool ADJ>
__device__ __forceinline__ Pairs<V> weights_at(const float* w, int c, int half) {
    float x[V], y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        x[i] = w[V * c + i];
        y[i] = w[half + V * c + i];
    }
    return pairs_of<V, ADJ>(x, y);
}

constexpr int kWidest = 512;

template <typename T, int LANES, int V, bool ADJ>
__global__ __launch_bounds__(kThreads, V == 8 ? 1 : kFwdPerSm) void fwd_kernel(Args a, Out o, int q_blocks) {
    // U heads in flight, two of them worked on at a time
    constexpr int GROUPS = kThreads / LANES, U = sizeof(T) == 2 ? kAhead : 2, P = V / 2;
    __shared__ __align__(16) float w[kWidest];
    const int half = a.D / 2;
    const bool lane_in = V * (threadIdx.x % LANES) < half;
    const int c = lane_in ? threadIdx.x % LANES : 0;
    const Share<T> s(a, q_blocks, GROUPS);
    T* dst = static_cast<T*>(s.is_k ? o.k : o.q) + V * c;
    int64_t j = s.first + threadIdx.x / LANES;
    Spot<T> at(s, j);
    Raw<T, V> rx[U], ry[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const T* x = at.x + (u < at.left ? u : 0) * s.s2 + V * c;
        rx[u] = load<V>(x);
        ry[u] = load<V>(x + half);
    }
    Angles<V> turn = angles_at<V, ADJ>(a, position(a, at.token), c);
    for (int d = threadIdx.x; d < a.D; d += kThreads)
        w[d] = weight_at<float>(s.is_k ? a.wk : a.wq, a.w_dtype, d);
    __syncthreads();
    const float inv_d = 1.f / a.D, eps = static_cast<float>(a.eps);
    // all lanes of the block make the same number of rounds
    for (int64_t j0 = s.first; j0 < s.jobs; j0 += s.step) {
        // the weights go into the cosines and sines of a token
        float2 uc[P], us[P], vc[P], vs[P];
        const Pairs<V> wp = weights_at<V, ADJ>(w, c, half);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            uc[i] = __fmul2_rn(wp.u[i], turn.c[i]);
            us[i] = __fmul2_rn(wp.u[i], turn.s[i]);
            vc[i] = __fmul2_rn(wp.v[i], turn.c[i]);
            vs[i] = neg(__fmul2_rn(wp.v[i], turn.s[i]));
        }
        j += s.step;
        const Spot<T> next(s, j);
        turn = angles_at<V, ADJ>(a, position(a, next.token), c);
        for (int r = 0; r < s.per; r += U) {
            const Spot<T> then = r + U >= s.per ? next : at.after(s, U);
#pragma unroll
            for (int u0 = 0; u0 < U; u0 += 2) {
                Pairs<V> x[2];
                float sq[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int u = u0 + k;
                    x[k] = unpack<ADJ>(rx[u], ry[u]);
                    const T* from = then.x + (u < then.left ? u : 0) * s.s2 + V * c;
                    rx[u] = load<V>(from);
                    ry[u] = load<V>(from + half);
                    float2 q = __fmul2_rn(x[k].u[0], x[k].u[0]);
                    q = __ffma2_rn(x[k].v[0], x[k].v[0], q);
#pragma unroll
                    for (int i = 1; i < P; ++i) {
                        q = __ffma2_rn(x[k].u[i], x[k].u[i], q);
                        q = __ffma2_rn(x[k].v[i], x[k].v[i], q);
                    }
                    sq[k] = lane_in ? q.x + q.y : 0.f;
                }
                group_sums<LANES>(sq);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float2 rn = twice(rsqrtf(sq[k] * inv_d + eps));
                    Pairs<V> y;
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        const float2 p = __fmul2_rn(x[k].u[i], rn), q = __fmul2_rn(x[k].v[i], rn);
                        y.u[i] = __ffma2_rn(p, uc[i], __fmul2_rn(q, vs[i]));
                        y.v[i] = __ffma2_rn(p, us[i], __fmul2_rn(q, vc[i]));
                    }
                    if (lane_in && u0 + k < at.left)
                        store<ADJ>(dst + (at.row + u0 + k) * a.D, half, y);
                }
            }
            at = then;
        }
    }
}

template <typename T, int LANES, int V, bool ADJ>
__global__ __launch_bounds__(kThreads, V == 8 ? 1 : kBwdPerSm) void bwd_kernel(Args a, Grad g, int q_blocks) {
    constexpr int GROUPS = kThreads / LANES, U = sizeof(T) == 2 ? kAhead : 2, P = V / 2;
    constexpr int WARPS = kThreads / 32;
    __shared__ __align__(16) float w[kWidest];
    __shared__ float sums[WARPS][2 * V * LANES];
    const int half = a.D / 2;
    const bool lane_in = V * (threadIdx.x % LANES) < half;
    const int c = lane_in ? threadIdx.x % LANES : 0;
    const Share<T> s(a, q_blocks, GROUPS);
    const T* gsrc = static_cast<const T*>(s.is_k ? g.gk : g.gq) + V * c;
    T* dst = static_cast<T*>(s.is_k ? g.dk : g.dq) + V * c;
    int64_t j = s.first + threadIdx.x / LANES;
    Spot<T> at(s, j);
    Raw<T, V> rx[U], ry[U], rg[U], ri[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int h = u < at.left ? u : 0;
        const T *x = at.x + h * s.s2 + V * c, *y = gsrc + (at.row + h) * a.D;
        rx[u] = load<V>(x);
        ry[u] = load<V>(x + half);
        rg[u] = load<V>(y);
        ri[u] = load<V>(y + half);
    }
    Angles<V> turn = angles_at<V, ADJ>(a, position(a, at.token), c);
    for (int d = threadIdx.x; d < a.D; d += kThreads)
        w[d] = weight_at<float>(s.is_k ? a.wk : a.wq, a.w_dtype, d);
    __syncthreads();
    const Pairs<V> wp = weights_at<V, ADJ>(w, c, half);
    Pairs<V> dw;
#pragma unroll
    for (int i = 0; i < P; ++i) dw.u[i] = dw.v[i] = twice(0.f);
    const float inv_d = 1.f / a.D, eps = static_cast<float>(a.eps);
    for (int64_t j0 = s.first; j0 < s.jobs; j0 += s.step) {
        j += s.step;
        const Spot<T> next(s, j);
        const Angles<V> turn_next = angles_at<V, ADJ>(a, position(a, next.token), c);
        for (int r = 0; r < s.per; r += U) {
            const Spot<T> then = r + U >= s.per ? next : at.after(s, U);
#pragma unroll
            for (int u0 = 0; u0 < U; u0 += 2) {
                Pairs<V> x[2], h[2];
                float part[4];   // of both heads: squares, then products
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int u = u0 + k;
                    x[k] = unpack<ADJ>(rx[u], ry[u]);
                    const Pairs<V> y = unpack<ADJ>(rg[u], ri[u]);
                    const int hd = u < then.left ? u : 0;
                    const T *from = then.x + hd * s.s2 + V * c, *gfrom = gsrc + (then.row + hd) * a.D;
                    rx[u] = load<V>(from);
                    ry[u] = load<V>(from + half);
                    rg[u] = load<V>(gfrom);
                    ri[u] = load<V>(gfrom + half);
                    float2 q = twice(0.f), dot = twice(0.f);
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        q = __ffma2_rn(x[k].u[i], x[k].u[i], q);
                        q = __ffma2_rn(x[k].v[i], x[k].v[i], q);
                        // turned back
                        h[k].u[i] = __ffma2_rn(y.u[i], turn.c[i], __fmul2_rn(y.v[i], turn.s[i]));
                        h[k].v[i] = __ffma2_rn(y.v[i], turn.c[i], __fmul2_rn(y.u[i], neg(turn.s[i])));
                        dot = __ffma2_rn(__fmul2_rn(h[k].u[i], wp.u[i]), x[k].u[i], dot);
                        dot = __ffma2_rn(__fmul2_rn(h[k].v[i], wp.v[i]), x[k].v[i], dot);
                    }
                    part[k] = lane_in ? q.x + q.y : 0.f;
                    part[2 + k] = lane_in ? dot.x + dot.y : 0.f;
                }
                group_sums<LANES>(part);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (!lane_in || u0 + k >= at.left) continue;
                    const float rn = rsqrtf(part[k] * inv_d + eps);
                    const float2 r2 = twice(rn), f = twice(-rn * rn * rn * part[2 + k] * inv_d);
                    Pairs<V> dx;
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        const float2 p = __fmul2_rn(h[k].u[i], r2), q = __fmul2_rn(h[k].v[i], r2);
                        dw.u[i] = __ffma2_rn(p, x[k].u[i], dw.u[i]);
                        dw.v[i] = __ffma2_rn(q, x[k].v[i], dw.v[i]);
                        dx.u[i] = __ffma2_rn(p, wp.u[i], __fmul2_rn(x[k].u[i], f));
                        dx.v[i] = __ffma2_rn(q, wp.v[i], __fmul2_rn(x[k].v[i], f));
                    }
                    store<ADJ>(dst + (at.row + u0 + k) * a.D, half, dx);
                }
            }
            at = then;
        }
        turn = turn_next;
    }
    if (!g.want_w) return;
    // groups of a warp, then the warps, in a fixed order
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) {
        const float2 t = i < V ? dw.u[i / 2] : dw.v[(i - V) / 2];
        float v = i % 2 ? t.y : t.x;
#pragma unroll
        for (int m = LANES; m < 32; m <<= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
        if (lane < LANES) sums[warp][i * LANES + lane] = v;
    }
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += kThreads) {
        const int e = d < half ? d : d - half, in = e % V;   // channel of a lane's x or y
        const int i = ADJ ? (in % 2 ? V : 0) + (d < half ? 0 : V / 2) + in / 2 : (d < half ? 0 : V) + in;
        float v = 0;
        for (int k = 0; k < WARPS; ++k) v += sums[k][i * LANES + e / V];
        static_cast<float*>(g.part)[static_cast<int64_t>(blockIdx.x) * a.D + d] = v;
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

// Whether accesses of whole chunks serve this call: what it reads and writes lies in
// 16-byte units (a head of all others does when the first does: D is a multiple of 8).
bool wide(const nsc_norm_rotate* a, const Out* o, const Grad* g) {
    if (o && !(aligned16(o->q) && aligned16(o->k))) return false;
    if (g && !(aligned16(g->gq) && aligned16(g->gk) && aligned16(g->dq) && aligned16(g->dk)))
        return false;
    const int64_t es = dtype_size(a->dtype);
    // (fp64 would spill its two chunks; it takes the other kernel)
    bool w = a->dtype != NSC_F64 && a->D % 8 == 0 && (a->D <= 256 || a->D % 16 == 0) && a->rot_dim == a->D && a->rows > 0 && aligned16(a->q) &&
             aligned16(a->k);
    for (int i = 0; i < 3; ++i)
        w = w && a->q_stride[i] * es % 16 == 0 && a->k_stride[i] * es % 16 == 0;
    return w;
}

// (two chunks of four channels a lane, past 256 channels of eight)
int lanes_for(int D) {
    int n = 1;
    while (n * 8 < D && n < 32) n <<= 1;
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

template <typename T, int LANES, int V = 4>
nsc_status run_wide(Args a, const Out* o, const Grad* g, int* n_part, cudaStream_t st) {
    a.per = heads_per_job(a, LANES);
    const int nq = (a.Hq + a.per - 1) / a.per, nk = (a.Hkv + a.per - 1) / a.per;
    // blocks of q and of k in the ratio of their work, as many as are resident at most
    constexpr int groups = kThreads / LANES;
    const int64_t most = 148 * (V == 8 ? 1 : o ? kFwdPerSm : kBwdPerSm);
    int64_t bq = (a.tokens * nq + groups - 1) / groups, bk = (a.tokens * nk + groups - 1) / groups;
    if (bq + bk > most) {
        const int64_t all = static_cast<int64_t>(a.Hq) + a.Hkv;
        bk = a.Hkv ? (most * static_cast<int64_t>(a.Hkv) + all - 1) / all : 0;
        bq = most - bk;
        if (a.Hq && bq < 1) { bq = 1; bk = most - 1; }
    }
    const unsigned blocks = static_cast<unsigned>(bq + bk);
    if (o) {
        auto kern = a.adjacent ? fwd_kernel<T, LANES, V, true> : fwd_kernel<T, LANES, V, false>;
        kern<<<blocks, kThreads, 0, st>>>(a, *o, static_cast<int>(bq));
        return check_launch("qk_norm_rotate");
    }
    n_part[0] = static_cast<int>(bq);
    n_part[1] = static_cast<int>(bq + bk);
    auto kern = a.adjacent ? bwd_kernel<T, LANES, V, true> : bwd_kernel<T, LANES, V, false>;
    kern<<<blocks, kThreads, 0, st>>>(a, *g, n_part[0]);
    return check_launch("qk_norm_rotate backward");
}

template <typename T, typename A>
nsc_status run(const nsc_norm_rotate* n, const Out* o, const Grad* g, int* n_part,
               cudaStream_t st) {
    Args a = args(n);
    if constexpr (sizeof(T) < 8) if (wide(n, o, g)) {
        switch (lanes_for(a.D)) {
            case 1: return run_wide<T, 1>(a, o, g, n_part, st);
            case 2: return run_wide<T, 2>(a, o, g, n_part, st);
            case 4: return run_wide<T, 4>(a, o, g, n_part, st);
            case 8: return run_wide<T, 8>(a, o, g, n_part, st);
            case 16: return run_wide<T, 16>(a, o, g, n_part, st);
            default:
                return a.D <= 256 ? run_wide<T, 32>(a, o, g, n_part, st)
                                  : run_wide<T, 32, 8>(a, o, g, n_part, st);
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
    auto kern = any_kernel<T, A>;
    const nsc_status ready = raise_shared("qk_norm_rotate", reinterpret_cast<const void*>(kern), smem);
    if (ready != NSC_OK) return ready;
    kern<<<static_cast<unsigned>(blocks), kThreads, smem, st>>>(
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
