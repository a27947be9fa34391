// capi.cu -- ABI marker, version and error reporting of libnsc_b200.so.
#include <mutex>
#include <string>
#include <unordered_map>

#include "nsc_host.h"

namespace nsc {
std::string& last_error() {
    thread_local std::string msg;
    return msg;
}

nsc_status raise_shared(const char* op, const void* kern, size_t bytes, int threads, int registers) {
    static std::mutex mu;
    static std::unordered_map<uint64_t, size_t> limits;   // of (kernel, device), as set so far
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess)
        return fail(NSC_ERR_LAUNCH_FAILED, "%s: no current device", op);
    const uint64_t key = reinterpret_cast<uint64_t>(kern) * 64 + static_cast<uint64_t>(dev);
    std::lock_guard<std::mutex> lock(mu);
    const auto hit = limits.find(key);
    if (hit != limits.end() && hit->second >= bytes) return NSC_OK;
    cudaFuncAttributes at{};
    if (cudaFuncGetAttributes(&at, kern) != cudaSuccess)
        return fail(NSC_ERR_LAUNCH_FAILED, "%s: kernel is not available: %s", op,
                    cudaGetErrorString(cudaGetLastError()));
    if (at.numRegs * threads < registers)
        return fail(NSC_ERR_LAUNCH_FAILED, "%s: kernel holds %d registers a thread", op, at.numRegs);
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(bytes)) != cudaSuccess)
        return fail(NSC_ERR_LAUNCH_FAILED, "%s: %zu bytes of shared memory: %s", op, bytes,
                    cudaGetErrorString(cudaGetLastError()));
    limits[key] = bytes;
    return NSC_OK;
}
}  // namespace nsc

extern "C" {

int nsc_index_width_bits(void) { return 64; }

const char* nsc_version(void) { return "0.12.0-b200.1"; }

const char* nsc_last_error_string(void) { return nsc::last_error().c_str(); }

}  // extern "C"
