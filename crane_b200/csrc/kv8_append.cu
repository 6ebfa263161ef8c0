// Rows of keys and values into the pages of an 8-bit cache (kv8.cuh).
//
// A page and head of keys or of values has one scale, the smallest power of two 2^e with max |y| <= 448 2^e over the rows it was given since its first position
// was written (max |y| counts as 2^-100 at least); code = e4m3(y / 2^e), to nearest even.  A page that is continued takes the larger of its own scale and the new
// rows': dividing its codes by a power of two is exact but for those that become subnormal, so rows that came in one by one have the codes they would have had
// together, up to that.  With scales that are not powers of two each growth would round every code of the page again.
// Infinities become NaN (e4m3 has none) and leave the scale alone; NaN stays NaN.
//
// Bound by bytes for prompts, by latency for single tokens.  One CTA takes what a page and head of keys, or of values, gets: no other one writes there.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "kv8.cuh"

namespace cb {
namespace {

constexpr int AP_THREADS = 128;

__device__ __forceinline__ float ld1(const void* p, int type, long long i) {
    if (type == KV8_F32) return __ldg(reinterpret_cast<const float*>(p) + i);
    const unsigned short u = __ldg(reinterpret_cast<const unsigned short*>(p) + i);
    return type == KV8_BF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
}
// Eight columns; VEC: aligned to 16 bytes
template <bool VEC>
__device__ __forceinline__ void ld8(const void* p, int type, long long i, float* y) {
    if constexpr (VEC) {
        if (type == KV8_F32) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i));
            const float4 b = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i) + 1);
            y[0] = a.x; y[1] = a.y; y[2] = a.z; y[3] = a.w; y[4] = b.x; y[5] = b.y; y[6] = b.z; y[7] = b.w;
            return;
        }
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned short*>(p) + i));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (type == KV8_BF16) { y[2 * j] = bf16lo(w[j]); y[2 * j + 1] = bf16hi(w[j]); }
            else { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j])); y[2 * j] = f.x; y[2 * j + 1] = f.y; }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = ld1(p, type, i + j);
    }
}
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
template <bool VEC, bool BY_ROW>
__global__ void __launch_bounds__(AP_THREADS)
append_kernel(Kv8Rows kr, Kv8Rows vr, Kv8Pool pool, Kv8Seqs s) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float wmax[AP_THREADS / 32];
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
    const int cpr = D / 8, total = count * cpr, kept = pos - block * P;
    float top = 0.f;
    for (int c = tid; c < total; c += AP_THREADS) {
        float y[8];
        const int r = c / cpr;
        ld8<VEC>(x.p, x.type, base + r * x.ld + (c - r * cpr) * 8, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) if (!infinite(y[j])) top = fmaxf(top, fabsf(y[j]));
    }
    top = warp_max(top);
    if ((tid & 31) == 0) wmax[tid >> 5] = top;
    float* sp = pool.scales + ((size_t)page * pool.kv_heads + head) * 2 + half;
    const float own = kept ? *sp : 0.f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < AP_THREADS / 32; ++w) top = fmaxf(top, wmax[w]);
    top = fmaxf(top, 0x1p-100f);
    const uint32_t bits = __float_as_uint(top);                      // top = m 2^(E - 127), m in [1, 2); 448 = 1.75 x 2^8
    const uint32_t e = (bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
    const float scale = fmaxf(__uint_as_float(e << 23), own);
    const float inv = __frcp_rn(scale);
    unsigned char* dst = (half ? pool.v : pool.k) + ((size_t)page * pool.kv_heads + head) * P * D;
    if (kept && scale != own) {                                      // (uniform in the CTA)
        const float ratio = own * inv;
        for (int c = tid; c < kept * D / 8; c += AP_THREADS) {
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
    for (int c = tid; c < total; c += AP_THREADS) {
        float y[8];
        const int r = c / cpr;
        ld8<VEC>(x.p, x.type, base + r * x.ld + (c - r * cpr) * 8, y);
        uint2 u;
        uint32_t* w = &u.x;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t v = 0;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float a = y[4 * i + 2 * j], c2 = y[4 * i + 2 * j + 1];
                v |= codes2(infinite(a) ? NAN : a * inv, infinite(c2) ? NAN : c2 * inv) << (16 * j);
            }
            w[i] = v;
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
    auto f = vec ? (by_row ? append_kernel<true, true> : append_kernel<true, false>) : (by_row ? append_kernel<false, true> : append_kernel<false, false>);
    return launch_k(f, grid, dim3(AP_THREADS), 0, st, pdl, k, v, pool, s);
}

}  // namespace cb
