// token_attention_tc.cu -- host side of the tensor-core token-attention kernels:
// which calls they take, tensor maps, shared-memory and register checks.
#include <cudaTypedefs.h>

#include <mutex>
#include <unordered_map>

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

bool aligned(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; }

bool boxable(const int64_t* s, int B, int L, int H) {
    const int n[3] = {B, L, H};
    for (int i = 0; i < 3; ++i)
        if (n[i] > 1 && (s[i] <= 0 || s[i] % 8 || s[i] >= (1LL << 38))) return false;
    return true;
}

}  // namespace

bool encode_heads(CUtensorMap* map, const void* base, const int64_t* strides, int B, int L, int H,
                  int D, bool bf16, const char** err) {
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
    const cuuint32_t box[4] = {64, 1, kRows, 1}, one[4] = {1, 1, 1, 1};
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

nsc_status tc_ready(const void* kern, int smem, int threads, int registers) {
    // the largest shared memory asked for so far of (device, kernel)
    static std::mutex mu;
    static std::unordered_map<uint64_t, int> asked;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess)
        return fail(NSC_ERR_LAUNCH_FAILED, "token_attention: no current device");
    const uint64_t key = reinterpret_cast<uint64_t>(kern) * 64 + static_cast<uint64_t>(dev);
    std::lock_guard<std::mutex> lock(mu);
    auto hit = asked.find(key);
    if (hit != asked.end() && hit->second >= smem) return NSC_OK;
    cudaFuncAttributes at{};
    if (cudaFuncGetAttributes(&at, kern) != cudaSuccess)
        return fail(NSC_ERR_LAUNCH_FAILED, "token_attention: kernel is not available");
    if (at.numRegs * threads < registers)
        return fail(NSC_ERR_LAUNCH_FAILED, "token_attention: kernel holds %d registers a thread",
                    at.numRegs);
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
        cudaSuccess)
        return fail(NSC_ERR_LAUNCH_FAILED, "token_attention: %d bytes of shared memory", smem);
    asked[key] = smem;
    return NSC_OK;
}

bool tc_fits(const Params& p, int dtype) {
    return (dtype == NSC_F16 || dtype == NSC_BF16) && p.D % 8 == 0 && p.D <= 128 && p.Lk > 0 &&
           !p.lengths && p.scale > 0 && aligned(p.q) && aligned(p.k) && aligned(p.v) &&
           boxable(p.qs, p.B, p.Lq, p.Hq) && boxable(p.ks, p.B, p.Lk, p.Hkv) &&
           boxable(p.vs, p.B, p.Lk, p.Hkv);
}

nsc_status tc_fwd(const Params& p, int dtype, cudaStream_t st) {
    if (dtype == NSC_BF16)
        return p.D <= 64 ? tc_fwd_run<__nv_bfloat16, 64>(p, st)
                         : tc_fwd_run<__nv_bfloat16, 128>(p, st);
    return p.D <= 64 ? tc_fwd_run<__half, 64>(p, st) : tc_fwd_run<__half, 128>(p, st);
}

}  // namespace tok
}  // namespace nsc
