// token_warp_mma.cuh -- warp-wide 16-bit products (16 rows by 8 columns by 16) and
// asynchronous copies, for the token-attention kernels whose tiles are too small for
// the 128 rows of a tcgen05 product.
#pragma once

#include <type_traits>

#include "nsc_tcgen05.cuh"
#include "token_attention.h"

namespace nsc {
namespace tok {

// tanh y to some 4e-7 of itself: below |y| = 0.25 by its series, whose next term is 2.2e-2 y^8
// of the sum (3e-7), since 1 - 2 / (1 + e^(2|y|)) is good to 1e-7 of one only: with a cap in the
// thousands, of which scores are a small part, that is 1e-3 of a score and more.
__device__ __forceinline__ float tanh_exact(float y) {
    const float e = tc::ex2(fabsf(y) * static_cast<float>(2 * kLog2e)), u = y * y;
    float p = fmaf(u, -17.f / 315.f, 2.f / 15.f);
    p = fmaf(p, u, -1.f / 3.f);
    p = fmaf(p * u, y, y);
    return fabsf(y) < 0.25f ? p : copysignf(1.f - __fdividef(2.f, 1.f + e), y);
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? 16 : 0;
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(n)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() {
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N> __device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, "
                     "{%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, "
                     "{%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

}  // namespace tok
}  // namespace nsc
