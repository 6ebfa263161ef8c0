// Host test of crane_b200/csrc/smem_optin.h against a fake of the CUDA calls it makes: two threads whose first launches of a kernel want different sizes; whatever their order, a launch
// finds an attribute as large as it asked for.
#include "../../crane_b200/csrc/smem_optin.h"

#include <chrono>
#include <cstdio>
#include <thread>

static std::atomic<int> attribute{0}, calls{0}, inside{0};
static cudaError_t set_attribute(int bytes) {
    const int n = ++calls;
    if (n == 1)                                      // the first waits for the other thread, as long as one can wait for it
        for (int i = 0; i < 200 && inside.load() < 2; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
    if (n == 1) std::this_thread::sleep_for(std::chrono::milliseconds(50));
    attribute = bytes;
    return cudaSuccess;
}
extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = 3; return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int bytes) { return set_attribute(bytes); }
}
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

int main() {
    static cb::SmemOptIn seen;
    const void* kernel = &seen;
    std::atomic<int> bad{0};
    auto launch = [&](size_t bytes) {
        ++inside;
        if (cb::ensure_dyn_smem(kernel, bytes, seen)) ++bad;
    };
    std::thread small([&] { launch(100000); });
    while (calls.load() == 0) std::this_thread::yield();
    std::thread large([&] { launch(200000); });
    small.join(); large.join();
    CHECK(bad == 0 && attribute == 200000 && seen.bytes[3] == 200000);
    const int n = calls;
    launch(150000); launch(200000);
    CHECK(calls == n && attribute == 200000);
    printf("smem_optin: ok\n");
    return 0;
}
