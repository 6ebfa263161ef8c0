// cudaFuncSetAttribute(MaxDynamicSharedMemorySize) is per DEVICE -- one process may drive a handle on every GPU of the box -- so each launcher remembers, per device, the largest
// opt-in it has already made for its kernel instantiation.  Several threads may launch at once.  Host code only.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <mutex>

namespace cb {

constexpr int CB_MAX_DEV = 64;
struct SmemOptIn { std::atomic<size_t> bytes[CB_MAX_DEV] = {}; };
inline std::mutex& smem_optin_mutex() { static std::mutex mu; return mu; }
template <typename K>
inline int ensure_dyn_smem(K kernel, size_t bytes, SmemOptIn& seen) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= CB_MAX_DEV) return (int)cudaErrorInvalidDevice;
    if (bytes <= seen.bytes[dev].load(std::memory_order_acquire)) return 0;
    std::lock_guard<std::mutex> g(smem_optin_mutex());             // (the attribute is what was set last: a smaller one must not come behind a larger)
    if (bytes <= seen.bytes[dev].load(std::memory_order_relaxed)) return 0;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) return (int)e;
    seen.bytes[dev].store(bytes, std::memory_order_release);
    return 0;
}

}  // namespace cb
