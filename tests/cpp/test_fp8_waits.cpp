// Host test of crane_b200/csrc/fp8_waits.h against a fake of the CUDA calls it makes: a raised word is reported to every stream once, whichever stream's work raised it, and stays where it is.
#include "../../crane_b200/csrc/fp8_waits.h"

#include <cstdio>
#include <cstdlib>
#include <thread>
#include <vector>

static int allocs = 0;
static bool fail_alloc = false;
static cudaStreamCaptureMode mode_now = cudaStreamCaptureModeGlobal;
extern "C" {
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaThreadExchangeStreamCaptureMode(cudaStreamCaptureMode* m) { std::swap(*m, mode_now); return cudaSuccess; }
cudaError_t cudaHostAlloc(void** p, size_t n, unsigned) {
    if (fail_alloc || mode_now != cudaStreamCaptureModeRelaxed) return cudaErrorMemoryAllocation;
    *p = malloc(n); *static_cast<int*>(*p) = 77; ++allocs; return cudaSuccess;
}
}
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

int main() {
    cb::F8Waits w;
    cudaStream_t a = (cudaStream_t)0x1000, b = (cudaStream_t)0x2000, c = (cudaStream_t)0x3000;
    CHECK(!w.take(a) && allocs == 0);                 // no linear yet
    fail_alloc = true;
    CHECK(w.word() == nullptr && mode_now == cudaStreamCaptureModeGlobal);
    fail_alloc = false;
    int* word = w.word();
    CHECK(word && *word == 0 && mode_now == cudaStreamCaptureModeGlobal);
    CHECK(!w.take(a) && !w.take(b));
    *word = 1;                                        // a graph captured on `a`, launched on `b`
    CHECK(w.take(b) && !w.take(b));
    CHECK(w.take(a) && !w.take(a) && !w.take(b));
    *word = 1;
    CHECK(w.take(a) && w.take(b) && w.take(c));       // c's first: it hears of all
    CHECK(!w.take(a) && !w.take(b) && !w.take(c));
    CHECK(w.word() == word && allocs == 1);
    cb::F8Waits many;
    std::vector<std::thread> t;
    std::vector<int*> got(8);
    for (int i = 0; i < 8; ++i) t.emplace_back([&, i] { got[i] = many.word(); });
    for (auto& x : t) x.join();
    for (int* p : got) CHECK(p && p == got[0]);
    CHECK(allocs == 2);
    printf("fp8_waits: ok\n");
    return 0;
}
