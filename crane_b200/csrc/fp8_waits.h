// Bounded waits that ran out in the linears of crane_b200_fp8_linear (TcWait, tc.cuh): one word a device, that every such kernel of it holds, and who has been told.  A linear that was
// captured runs on the stream that its graph is launched on, whichever that is, so a word of the stream that it was captured on would be looked at by nobody.  Host code only.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <mutex>
#include <unordered_map>

namespace cb {

class F8Waits {
public:
    // The current device's word, in pinned memory, made by the first call and never given back: captured graphs hold its address.  nullptr: no memory.
    int* word() {
        if (int* w = word_.load(std::memory_order_acquire)) return w;
        std::lock_guard<std::mutex> g(mu_);
        int* w = word_.load(std::memory_order_relaxed);
        if (w) return w;
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;       // (the stricter modes of a capture under way forbid its thread to pin memory)
        if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) { cudaGetLastError(); return nullptr; }
        if (cudaHostAlloc((void**)&w, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable) != cudaSuccess) { cudaGetLastError(); w = nullptr; }
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (!w) return nullptr;
        *w = 0;
        word_.store(w, std::memory_order_release);
        return w;
    }
    // True once a stream and time: a wait ran out, in whichever stream's work, since the last call for `st`, or ever if there was none.  The word does not say whose it was, so every
    // stream hears of it.  Called behind a synchronisation of `st`.
    bool take(cudaStream_t st) {
        int* w = word_.load(std::memory_order_acquire);
        if (!w) return false;
        std::lock_guard<std::mutex> g(mu_);
        if (__atomic_exchange_n(w, 0, __ATOMIC_ACQ_REL)) ++times_;
        if (!times_) return false;
        uint64_t& told = told_[st];
        const bool news = told != times_;
        told = times_;
        return news;
    }

private:
    std::atomic<int*> word_{nullptr};
    std::mutex mu_;
    uint64_t times_ = 0;                                                 // the word was found raised
    std::unordered_map<cudaStream_t, uint64_t> told_;                    // ... of those, what a stream has heard of (empty while no wait has run out)
};

}  // namespace cb
