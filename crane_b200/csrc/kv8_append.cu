// Rows of keys and values into the pages of an 8-bit cache (kv8.cuh).
//
// A page and head of keys or of values has one scale, the smallest power of two 2^e with max |y| <= 448 2^e over the rows it was given since its first position
// was written (max |y| counts as 2^-100 at least); code = e4m3(y / 2^e), to nearest even.  A page that is continued takes the larger of its own scale and the new
// rows': dividing its codes by a power of two is exact but for those that become subnormal, so rows that came in one by one have the codes they would have had
// together, up to that.  With scales that are not powers of two each growth would round every code of the page again.
// Infinities become NaN (e4m3 has none) and leave the scale alone; NaN stays NaN.
//
// Bound by bytes for prompts, by latency for single tokens.  One CTA takes what a page and head of keys, or of values, gets: no other one writes there.  Four prompts of 2048 tokens,
// 8 heads of 128, bf16: 48 MB in 13.7 us, 3.5 TB/s, five trips to the L2 one behind the other in 2 176 CTAs (read twice, in a loop, 20.5); a token of each of 64 sequences 3.5.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "kv8.cuh"

namespace cb {
namespace {

constexpr int CHUNKS = 8;                      // of eight columns that a thread has: a page and head stay in registers from their maximum to their codes

// Eight columns as they lie (VEC: on 16-byte boundaries), and as numbers
template <typename T> struct Eight {
    uint32_t w[2 * sizeof(T)];
    template <bool VEC> __device__ __forceinline__ void load(const T* p) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) { const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i); w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w; }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
        } else {
            const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __ldg(s + 2 * i) | (uint32_t)__ldg(s + 2 * i + 1) << 16;
        }
    }
    __device__ __forceinline__ float2 pair(int i) const {                    // columns 2 i and 2 i + 1
        if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[(2 * i) % (2 * sizeof(T))]), __uint_as_float(w[(2 * i + 1) % (2 * sizeof(T))]));
        else if constexpr (std::is_same<T, bf16>::value) return make_float2(bf16lo(w[i]), bf16hi(w[i]));
        else return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    }
};
__device__ __forceinline__ uint32_t codes2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ bool infinite(float v) { return fabsf(v) == INFINITY; }

// The largest b with key(b) <= at; key grows with b.  All lanes of a warp take part.
template <typename K>
__device__ __forceinline__ int search(int n, int at, K key) {
    int lo = 0;
    while (n > 1) {
        const int step = (n + 31) / 32, i = (int)(threadIdx.x & 31) * step;
        const unsigned m = __ballot_sync(0xffffffffu, i < n && key(lo + i) <= at);
        const int k = m ? 31 - __clz(m) : 0;
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}

// blockIdx.x: a piece (kv8_units.h)
template <typename T, int THREADS, bool VEC, bool BY_ROW>
__global__ void __launch_bounds__(THREADS)
append_kernel(Kv8Rows kr, Kv8Rows vr, Kv8Pool pool, Kv8Seqs s) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float wmax[THREADS / 32];
    const int P = pool.page, D = pool.dim, at = blockIdx.x, head = blockIdx.y, half = blockIdx.z, tid = threadIdx.x;
    const int b = search(s.seqs, at, [&](int i) { return kv8_piece_key(s, P, i, BY_ROW); });
    const Kv8Seq q = kv8_seq(s, b);
    const Kv8Piece piece = kv8_piece(s, q, P, b, at, BY_ROW);
    const int block = piece.block, pos = piece.pos, count = piece.count;
    if (!count) return;
    const int page = kv8_page(s, pool, b, block);
    if (page < 0) return;
    const Kv8Rows& x = half ? vr : kr;
    const long long base = (long long)(q.s0 + pos - q.first) * x.ld + (long long)head * x.ldh;
    const int cpr = D / 8, total = count * cpr, kept = pos - block * P;      // (at most THREADS * CHUNKS)
    float top = 0.f;
    Eight<T> y[CHUNKS];
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        const int c = tid + i * THREADS, row = c / cpr;
        if (c < total) y[i].template load<VEC>(reinterpret_cast<const T*>(x.p) + base + row * x.ld + (c - row * cpr) * 8);
    }
    float* sp = pool.scales + ((size_t)page * pool.kv_heads + head) * 2 + half;
    const float own = kept ? *sp : 0.f;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
        if (tid + i * THREADS < total)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 v = y[i].pair(j);
                if (!infinite(v.x)) top = fmaxf(top, fabsf(v.x));
                if (!infinite(v.y)) top = fmaxf(top, fabsf(v.y));
            }
    top = warp_max(top);
    if ((tid & 31) == 0) wmax[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) top = fmaxf(top, wmax[w]);
    top = fmaxf(top, 0x1p-100f);
    const uint32_t bits = __float_as_uint(top);                      // top = m 2^(E - 127), m in [1, 2); 448 = 1.75 x 2^8
    const uint32_t e = (bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
    const float scale = fmaxf(__uint_as_float(e << 23), own);
    const float inv = __frcp_rn(scale);
    unsigned char* dst = (half ? pool.v : pool.k) + ((size_t)page * pool.kv_heads + head) * P * D;
    if (kept && scale != own) {                                      // (uniform in the CTA)
        const float ratio = own * inv;
        for (int c = tid; c < kept * D / 8; c += THREADS) {
            uint2* p = reinterpret_cast<uint2*>(dst) + c;
            uint2 u = *p;
            uint32_t* w = &u.x;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t old = w[i];
                uint32_t now = 0;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(old >> (16 * j)), __NV_E4M3);
                    const float2 f = __half22float2(__half2(h));
                    now |= codes2(f.x * ratio, f.y * ratio) << (16 * j);
                }
                w[i] = now;
            }
            *p = u;
        }
    }
    dst += (size_t)kept * D;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        const int c = tid + i * THREADS;
        if (c >= total) break;
        uint2 u;
        uint32_t* w = &u.x;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 v = y[i].pair(k);
            const uint32_t two = codes2(infinite(v.x) ? NAN : v.x * inv, infinite(v.y) ? NAN : v.y * inv);
            if (k & 1) w[k >> 1] |= two << 16;
            else w[k >> 1] = two;
        }
        reinterpret_cast<uint2*>(dst)[c] = u;
    }
    if (tid == 0 && (!kept || scale != own)) *sp = scale;
}

bool vec_ok(const Kv8Rows& r) {
    const int per = r.type == KV8_F32 ? 4 : 8;
    return reinterpret_cast<uintptr_t>(r.p) % 16 == 0 && r.ld % per == 0 && r.ldh % per == 0;
}

}  // namespace

int kv8_append_launch(cudaStream_t st, const Kv8Rows& k, const Kv8Rows& v, const Kv8Pool& pool, const Kv8Seqs& s, bool pdl) {
    if (s.rows == 0 || s.seqs == 0) return 0;
    const long long slots = (long long)s.rows / pool.page + 2LL * s.seqs;
    const bool vec = vec_ok(k) && vec_ok(v), by_row = s.rows <= slots;
    const dim3 grid((unsigned)(by_row ? s.rows : slots), pool.kv_heads, 2);
    const int threads = pool.page * pool.dim / (8 * CHUNKS);
    auto go = [&](auto type, auto count) {
        using T = decltype(type);
        constexpr int N = decltype(count)::value;
        auto f = vec ? (by_row ? append_kernel<T, N, true, true> : append_kernel<T, N, true, false>) : (by_row ? append_kernel<T, N, false, true> : append_kernel<T, N, false, false>);
        return launch_k(f, grid, dim3(N), 0, st, pdl, k, v, pool, s);
    };
    auto sized = [&](auto type) {
        if (threads <= 128) return go(type, std::integral_constant<int, 128>());
        return threads == 256 ? go(type, std::integral_constant<int, 256>()) : go(type, std::integral_constant<int, 512>());
    };
    return k.type == KV8_F32 ? sized(float()) : k.type == KV8_BF16 ? sized(bf16()) : sized(__half());
}

}  // namespace cb
