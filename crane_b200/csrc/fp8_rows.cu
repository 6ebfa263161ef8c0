// Activation rows to e4m3 codes with a scale for every 128 columns: as they are, behind a gated unit, behind an RMS norm with the residual's addition.
//
//   a = max(max |y_k|, 2^-100) over the block's columns,  scale = a / 448,  code_k = e4m3(y_k * (448 / a))
//
// 448 is the largest e4m3 value, so the block's largest magnitude keeps all of its bits and nothing saturates but by the rounding of 448 / a; the bound keeps 448 / a
// finite (an empty block: codes 0).  The two divisions are f32, rounded to nearest; the code is the one rounding to 8 bits, to nearest even.  A NaN's code is NaN; an
// infinite magnitude makes its block's scale infinite and the block NaN wherever it is used.
//
// These kernels are bound by the bytes of the rows: one pass, a thread has 8 neighbouring columns (16 or 32 bytes in, 8 out) and 16 threads a block of 128, whose
// maximum takes four shuffles.
#include "fp8.cuh"

#include <cuda_fp16.h>

namespace cb {

constexpr float F8_TOP = 448.f;
constexpr float F8_TINY = 7.888609052210118e-31f;     // 2^-100

template <typename T> __device__ __forceinline__ float f8_float(T v);
template <> __device__ __forceinline__ float f8_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float f8_float<bf16>(bf16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float f8_float<__half>(__half v) { return __half2float(v); }

__device__ __forceinline__ void f8_unpack(const uint4& u, bf16, float* v) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = bf16lo(w[i]); v[2 * i + 1] = bf16hi(w[i]); }
}
__device__ __forceinline__ void f8_unpack(const uint4& u, __half, float* v) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
}
// columns c .. c + 7 of a row of K; zeros behind the last.  `vec`: whole chunks of the row lie on 16-byte boundaries
template <typename T>
__device__ __forceinline__ void f8_load8(const T* row, int c, int K, bool vec, float* v) {
    if (vec && c + 8 <= K) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            f8_unpack(*reinterpret_cast<const uint4*>(row + c), T(), v);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < K ? f8_float(row[c + i]) : 0.f;
    }
}
__device__ __forceinline__ void f8_load8(const void* base, int type, long long at, int c, int K, bool vec, float* v) {
    if (type == F8_F32) f8_load8(static_cast<const float*>(base) + at, c, K, vec, v);
    else if (type == F8_BF16) f8_load8(static_cast<const bf16*>(base) + at, c, K, vec, v);
    else f8_load8(static_cast<const __half*>(base) + at, c, K, vec, v);
}
// h = v rounded to the type, stored and given back in f32
template <typename T>
__device__ __forceinline__ void f8_store8(T* row, int c, int K, bool vec, float* v) {
    if constexpr (sizeof(T) == 4) {
        if (vec && c + 8 <= K) {
            *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(row + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) if (c + i < K) row[c + i] = v[i];
        }
    } else {
        T h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (std::is_same<T, bf16>::value) h[i] = __float2bfloat16_rn(v[i]); else h[i] = __float2half_rn(v[i]);
            v[i] = f8_float(h[i]);
        }
        if (vec && c + 8 <= K) *reinterpret_cast<uint4*>(row + c) = *reinterpret_cast<const uint4*>(h);
        else {
#pragma unroll
            for (int i = 0; i < 8; ++i) if (c + i < K) row[c + i] = h[i];
        }
    }
}
__device__ __forceinline__ void f8_store8(void* base, int type, long long at, int c, int K, bool vec, float* v) {
    if (type == F8_F32) f8_store8(static_cast<float*>(base) + at, c, K, vec, v);
    else if (type == F8_BF16) f8_store8(static_cast<bf16*>(base) + at, c, K, vec, v);
    else f8_store8(static_cast<__half*>(base) + at, c, K, vec, v);
}

__device__ __forceinline__ uint32_t f8_pair(float a, float b) {      // a in the low byte
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
// The block of 16 neighbouring threads (a half warp): scale and codes.  Every lane of the warp calls; `in`: this thread's columns c .. exist
__device__ __forceinline__ void f8_emit(const float* v, long long m, int c, int K, bool in, const F8Out& o) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(v[i]));
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, s));
    a = fmaxf(a, F8_TINY);
    const float inv = __fdiv_rn(F8_TOP, a);
    if (!in) return;
    if ((c & (F8_BLOCK - 1)) == 0) o.scales[(c / F8_BLOCK) * o.lds + m] = __fdiv_rn(a, F8_TOP);
    const uint32_t lo = f8_pair(v[0] * inv, v[1] * inv) | f8_pair(v[2] * inv, v[3] * inv) << 16, hi = f8_pair(v[4] * inv, v[5] * inv) | f8_pair(v[6] * inv, v[7] * inv) << 16;
    unsigned char* p = o.codes + m * o.ld + c;
    if (c + 8 <= K) *reinterpret_cast<uint2*>(p) = make_uint2(lo, hi);
    else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (c + i < K) p[i] = (unsigned char)((i < 4 ? lo : hi) >> (8 * (i & 3)));
    }
}

template <typename T, bool GATED>
__global__ void __launch_bounds__(256)
f8_rows_kernel(const T* __restrict__ x, long long ldx, long long M, int K, int KB, bool vec, F8Out o) {
    pdl_wait();
    pdl_launch_dependents();
    const long long g = (long long)blockIdx.x * 16 + (threadIdx.x >> 4), m = g / KB;
    const int c = (int)(g - m * KB) * F8_BLOCK + (threadIdx.x & 15) * 8;
    const bool in = m < M && c < K;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (in) {
        const T* row = x + m * ldx;
        f8_load8(row, c, K, vec, v);
        if constexpr (GATED) {
            float u[8];
            f8_load8(row + K, c, K, vec, u);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = silu_f(v[i]) * u[i];
        }
    }
    f8_emit(v, m, c, K, in, o);
}

struct F8NormArgs { F8Norm n; long long M; int K, tpr; bool vec_x, vec_r, vec_w; F8Out o; };
// `tpr` threads have a row (a block several, where it has fewer columns than 8 x 256), J chunks of 8 columns each, in registers between the sum and the codes; J = 0: any
// number, read again for the codes (what the thread itself stored, where there is a residual).
template <typename T, int J>
__global__ void __launch_bounds__(1024)
f8_norm_kernel(const F8NormArgs a) {
    __shared__ float red[32];
    const int t = threadIdx.x & (a.tpr - 1), lane = threadIdx.x & 31, warp = threadIdx.x >> 5, K = a.K;
    const long long m = (long long)blockIdx.x * (blockDim.x / a.tpr) + threadIdx.x / a.tpr;
    const bool row_in = m < a.M;
    const T* xr = static_cast<const T*>(a.n.x) + m * a.n.ldx;
    auto first = [&](int c, float* v) {                 // h of a chunk, stored where there is a residual
        if (!(row_in && c < K)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
            return;
        }
        f8_load8(xr, c, K, a.vec_x, v);
        if (a.n.residual) {
            float r[8];
            f8_load8(a.n.residual, a.n.res_type, m * a.n.ldr, c, K, a.vec_r, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += r[i];
            f8_store8(a.n.residual_out, a.n.res_type, m * a.n.ldr, c, K, a.vec_r, v);
        }
    };
    auto finish = [&](int c, float* v, float rstd) {
        const bool in = row_in && c < K;
        if (in) {
            float w[8];
            f8_load8(a.n.w, a.n.w_type, 0, c, K, a.vec_w, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * rstd * w[i];
        }
        f8_emit(v, m, c, K, in, a.o);
    };
    auto row_rstd = [&](float s) {
        s = warp_sum(s);
        if (a.tpr > 32) {
            const int nw = a.tpr >> 5, w0 = warp & ~(nw - 1);
            if (lane == 0) red[warp] = s;
            __syncthreads();
            s = warp_sum(lane < nw ? red[w0 + lane] : 0.f);
        }
        return rsqrtf(s / (float)K + a.n.eps);
    };
    pdl_wait();
    pdl_launch_dependents();
    float s = 0.f;
    if constexpr (J > 0) {
        float v[J][8];
#pragma unroll
        for (int j = 0; j < J; ++j) first((t + j * a.tpr) * 8, v[j]);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[j][i] * v[j][i];
        const float rstd = row_rstd(s);
#pragma unroll
        for (int j = 0; j < J; ++j) finish((t + j * a.tpr) * 8, v[j], rstd);
    } else {
        for (int c = t * 8; c < K; c += a.tpr * 8) {
            float v[8];
            first(c, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i] * v[i];
        }
        const float rstd = row_rstd(s);
        for (int c = t * 8; c < (K + 255) / 256 * 256; c += a.tpr * 8) {        // (a warp's threads leave the loop together)
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (row_in && c < K) {
                if (a.n.residual) f8_load8(a.n.residual_out, a.n.res_type, m * a.n.ldr, c, K, a.vec_r, v);
                else f8_load8(xr, c, K, a.vec_x, v);
            }
            finish(c, v, rstd);
        }
    }
}

static bool f8_aligned(const void* p, long long ld, int type) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * f8_bytes(type)) % 16 == 0; }

template <typename T, bool GATED>
static int f8_rows_t(cudaStream_t st, const void* x, int type, long long ldx, long long M, int K, const F8Out& out, bool pdl) {
    const int KB = f8_blocks(K);
    const long long blocks = (M * KB + 15) / 16;
    if (blocks > 0x7fffffffLL) return -1000;
    const bool vec = f8_aligned(x, ldx, type) && (!GATED || (long long)K * f8_bytes(type) % 16 == 0);
    return launch_k(f8_rows_kernel<T, GATED>, dim3((unsigned)blocks), dim3(256), 0, st, pdl, static_cast<const T*>(x), ldx, M, K, KB, vec, out);
}
template <bool GATED>
static int f8_rows_launch(cudaStream_t st, const void* x, int type, long long ldx, long long M, int K, const F8Out& out, bool pdl) {
    if (M == 0) return 0;
    switch (type) {
        case F8_F32:  return f8_rows_t<float, GATED>(st, x, type, ldx, M, K, out, pdl);
        case F8_BF16: return f8_rows_t<bf16, GATED>(st, x, type, ldx, M, K, out, pdl);
        case F8_F16:  return f8_rows_t<__half, GATED>(st, x, type, ldx, M, K, out, pdl);
        default: return -1000;
    }
}
int f8_quantize_launch(cudaStream_t st, const void* x, int type, long long ldx, long long M, int K, const F8Out& out, bool pdl) {
    return f8_rows_launch<false>(st, x, type, ldx, M, K, out, pdl);
}
int f8_silu_mul_launch(cudaStream_t st, const void* x, int type, long long ldx, long long M, int K, const F8Out& out, bool pdl) {
    return f8_rows_launch<true>(st, x, type, ldx, M, K, out, pdl);
}

template <typename T>
static int f8_norm_t(cudaStream_t st, F8NormArgs& a, bool pdl) {
    const int chunks = (a.K + 7) / 8;
    a.tpr = 32;
    while (a.tpr < 1024 && a.tpr < chunks) a.tpr *= 2;
    const int block = a.tpr < 256 ? 256 : a.tpr, rows = block / a.tpr;
    const long long blocks = (a.M + rows - 1) / rows;
    if (blocks > 0x7fffffffLL) return -1000;
    if (chunks <= a.tpr) return launch_k(f8_norm_kernel<T, 1>, dim3((unsigned)blocks), dim3(block), 0, st, pdl, a);
    if (chunks <= 2 * a.tpr) return launch_k(f8_norm_kernel<T, 2>, dim3((unsigned)blocks), dim3(block), 0, st, pdl, a);
    return launch_k(f8_norm_kernel<T, 0>, dim3((unsigned)blocks), dim3(block), 0, st, pdl, a);
}
int f8_rms_norm_launch(cudaStream_t st, const F8Norm& n, long long M, int K, const F8Out& out, bool pdl) {
    if (M == 0) return 0;
    F8NormArgs a = {n, M, K, 0, f8_aligned(n.x, n.ldx, n.type), n.residual && f8_aligned(n.residual, n.ldr, n.res_type) && f8_aligned(n.residual_out, n.ldr, n.res_type),
                    f8_aligned(n.w, 0, n.w_type), out};
    switch (n.type) {
        case F8_F32:  return f8_norm_t<float>(st, a, pdl);
        case F8_BF16: return f8_norm_t<bf16>(st, a, pdl);
        case F8_F16:  return f8_norm_t<__half>(st, a, pdl);
        default: return -1000;
    }
}

}  // namespace cb
