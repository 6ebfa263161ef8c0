// Activation rows to e4m3 codes with a scale for every 128 columns: as they are, behind a gated unit, behind an RMS norm with the residual's addition.
//
//   a = max(max |y_k|, 2^-100) over the block's columns,  scale = a / 448,  code_k = e4m3(y_k * (448 / a))
//
// 448 is the largest e4m3 value, so the block's largest magnitude keeps all of its bits and nothing saturates but by the rounding of 448 / a; the bound keeps 448 / a
// finite (an empty block: codes 0).  The two divisions are f32, rounded to nearest; the code is the one rounding to 8 bits, to nearest even.  A NaN's code is NaN; an
// infinite magnitude makes its block's scale infinite and the block NaN wherever it is used.
//
// These kernels are bound by the bytes of the rows, and next to them by instructions: one pass, a thread has 16 columns, 8 threads a block of 128, whose maximum takes three
// shuffles and whose two divisions are made eight times, not sixteen; as many blocks as the chip runs at once take rows in turn, with the next ones' loads on their way.
#include "fp8.cuh"

#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

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
// A thread has 16 columns of a block of 128, 8 from f8_col on and 8 from 64 behind those, 8 neighbouring threads the block.
__device__ __forceinline__ int f8_col(int thread) { return (thread >> 3) * F8_BLOCK + (thread & 7) * 8; }
// Rows on 16-byte boundaries (VEC) are read and written as that.  Others are read as the aligned pieces that hold them, of which the values are shifted out, and written one element at a
// time: there the eight threads of a block change values among themselves and take every eighth column, so that an instruction covers whole pieces of a row and not a value of each (all by elements, each thread its own: 8192 x 11001 to codes 113 us from f32, 70 from bf16, 583 f16 behind a norm
// with a residual; so 72, 67, 291).
__device__ __forceinline__ int f8_eighth(int c) { return (c & ~63) + ((c >> 3) & 7); }                   // the first of those, 8 to the next
// 8 threads' 8 values each, transposed: value i of thread t becomes value t of thread i.  Every lane calls
__device__ __forceinline__ void f8_turn(float* v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int b = 4; b > 0; b >>= 1) {
        const bool up = lane & b;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i & b) continue;
            const float got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + b], b);
            if (up) v[i] = got; else v[i + b] = got;
        }
    }
}
template <typename T>                              // 16-bit values
__device__ __forceinline__ void f8_turn(T* v) {
    const int lane = threadIdx.x & 31;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)*reinterpret_cast<const uint16_t*>(v + 2 * i) | (uint32_t)*reinterpret_cast<const uint16_t*>(v + 2 * i + 1) << 16;
#pragma unroll
    for (int b = 2; b > 0; b >>= 1) {
        const bool up = lane & (2 * b);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i & b) continue;
            const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? w[i] : w[i + b], 2 * b);
            if (up) w[i] = got; else w[i + b] = got;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = __byte_perm(w[i], __shfl_xor_sync(0xffffffffu, w[i], 1), lane & 1 ? 0x3276 : 0x5410);
        *reinterpret_cast<uint16_t*>(v + 2 * i) = (uint16_t)w[i]; *reinterpret_cast<uint16_t*>(v + 2 * i + 1) = (uint16_t)(w[i] >> 16);
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
// What a chunk brings, as it is loaded: to be asked for well ahead of its use, it must not be unpacked where it is loaded.  VEC: every chunk is whole and on its boundary.
template <typename T, bool VEC> struct F8Chunk {
    uint4 q[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* row, int c, int, bool in, const T*, const T*) {
        q[0] = in ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
        if constexpr (sizeof(T) == 4) q[1] = in ? *reinterpret_cast<const uint4*>(row + c + 4) : make_uint4(0, 0, 0, 0);
        else static_assert(sizeof(q) == 16, "one piece");
    }
    __device__ __forceinline__ void get(float* v, int, int) const {
        if constexpr (sizeof(T) == 4) {
            v[0] = __uint_as_float(q[0].x); v[1] = __uint_as_float(q[0].y); v[2] = __uint_as_float(q[0].z); v[3] = __uint_as_float(q[0].w);
            v[4] = __uint_as_float(q[1].x); v[5] = __uint_as_float(q[1].y); v[6] = __uint_as_float(q[1].z); v[7] = __uint_as_float(q[1].w);
        } else f8_unpack(q[0], T(), v);
    }
};
template <typename T> struct F8Chunk<T, false> {
    static constexpr int W = sizeof(T) == 4 ? 3 : 2;               // aligned pieces that hold 8 values
    uint4 q[W];
    int s;                                                         // bytes ahead of the values
    // Pieces that hold a byte of the row: what else is in them, between two rows or of the next, is shifted out.  `first`, `end`: of all rows, nothing outside of these is read
    __device__ __forceinline__ void load(const T* row, int c, int K, bool in, const T* first, const T* end) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(row + c), w = at & ~(uintptr_t)15;
        s = (int)(at & 15);
        if (!in) {
#pragma unroll
            for (int j = 0; j < W; ++j) q[j] = make_uint4(0, 0, 0, 0);
        } else if (w >= reinterpret_cast<uintptr_t>(first) && w + 16 * W <= reinterpret_cast<uintptr_t>(end)) {
#pragma unroll
            for (int j = 0; j < W; ++j) q[j] = j == 0 || w + 16 * j < reinterpret_cast<uintptr_t>(row + K) ? reinterpret_cast<const uint4*>(w)[j] : make_uint4(0, 0, 0, 0);
        } else {
            alignas(16) T t[16 * W / sizeof(T)];
#pragma unroll
            for (int j = 0; j < 16 * W / (int)sizeof(T); ++j) {
                const T* p = reinterpret_cast<const T*>(w) + j;
                t[j] = p >= row && p < row + K ? *p : T(0.f);
            }
#pragma unroll
            for (int j = 0; j < W; ++j) q[j] = reinterpret_cast<const uint4*>(t)[j];
        }
    }
    __device__ __forceinline__ void get(float* v, int c, int K) const {
        uint32_t w[4 * W];
#pragma unroll
        for (int j = 0; j < W; ++j) { w[4 * j] = q[j].x; w[4 * j + 1] = q[j].y; w[4 * j + 2] = q[j].z; w[4 * j + 3] = q[j].w; }
        constexpr int N = 2 * (int)sizeof(T);                      // words of 8 values
#pragma unroll
        for (int j = 0; j < N + 2 && j + 2 < 4 * W; ++j) w[j] = s & 8 ? w[j + 2] : w[j];
#pragma unroll
        for (int j = 0; j < N + 1 && j + 1 < 4 * W; ++j) w[j] = s & 4 ? w[j + 1] : w[j];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
        } else {
            const uint32_t by = s & 2 ? 0x5432 : 0x3210;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = __byte_perm(w[j], w[j + 1], by);
            f8_unpack(make_uint4(w[0], w[1], w[2], w[3]), T(), v);
        }
        if (c + 8 > K) {
#pragma unroll
            for (int i = 0; i < 8; ++i) if (c + i >= K) v[i] = 0.f;
        }
    }
};
// h = v rounded to the type, stored where the row is one and given back in f32.  Every lane calls
template <typename T, bool VEC>
__device__ __forceinline__ void f8_store8(T* row, int c, int K, bool row_in, float* v) {
    alignas(16) T h[8];
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = v[i];
    } else {                                    // two at a time, as the instruction has them
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            if constexpr (std::is_same<T, bf16>::value) {
                const uint32_t u = pack_bf16(v[i], v[i + 1]);
                *reinterpret_cast<uint32_t*>(h + i) = u;
                v[i] = bf16lo(u); v[i + 1] = bf16hi(u);
            } else {
                const __half2 u = __floats2half2_rn(v[i], v[i + 1]);
                *reinterpret_cast<__half2*>(h + i) = u;
                const float2 f = __half22float2(u);
                v[i] = f.x; v[i + 1] = f.y;
            }
        }
    }
    if constexpr (VEC) {
        if (!row_in || c >= K) return;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(row + c)[i] = reinterpret_cast<const uint4*>(h)[i];
    } else {
        f8_turn(h);
#pragma unroll
        for (int i = 0; i < 8; ++i) if (row_in && f8_eighth(c) + 8 * i < K) row[f8_eighth(c) + 8 * i] = h[i];
    }
}

__device__ __forceinline__ uint32_t f8_quad(float a, float b, float c, float d) {      // a in the low byte
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};\n\t}" : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}
// Scale and codes of a thread's 16 columns.  Every lane of the warp calls
template <bool VEC>
__device__ __forceinline__ void f8_emit(const float (*v)[8], long long m, int c, int K, bool row_in, const F8Out& o) {
    float a = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(v[h][i]));
#pragma unroll
    for (int s = 4; s > 0; s >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, s));
    a = fmaxf(a, F8_TINY);
    const float inv = __fdiv_rn(F8_TOP, a);
    if (!row_in || c >= K) return;
    if ((c & (F8_BLOCK - 1)) == 0) o.scales[(c / F8_BLOCK) * o.lds + m] = __fdiv_rn(a, F8_TOP);
    unsigned char* p = o.codes + m * o.ld + c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t lo = f8_quad(v[h][0] * inv, v[h][1] * inv, v[h][2] * inv, v[h][3] * inv), hi = f8_quad(v[h][4] * inv, v[h][5] * inv, v[h][6] * inv, v[h][7] * inv);
        const int at = c + 64 * h;
        if (VEC ? at < K : at + 8 <= K) *reinterpret_cast<uint2*>(p + 64 * h) = make_uint2(lo, hi);
        else if (!VEC) {
#pragma unroll
            for (int i = 0; i < 8; ++i) if (at + i < K) p[64 * h + i] = (unsigned char)((i < 4 ? lo : hi) >> (8 * (i & 3)));
        }
    }
}

// SiLU(g) u = g / (1 + z) u, z = exp(-g).  z / 4 = 2^(t - 2), t = -g log2 e, what t's rounding lost (lo) made good to first order; 4 / (1 + z) by rcp.approx, which an infinite gate stays
// infinite through.  By quarters, because 1 / (1 + z) would leave the normal numbers, where the reciprocal gives zero, ahead of g / (1 + z); where z itself passes 2^128 (g < -88.72) it
// does, and the result is zero.  The exponent's g is held to -90 .. 88: above, z vanishes against 1.
// Fourteen instructions and errors to five ulp (measured over -88.7 .. 88; four with a step of Newton's on the reciprocal), as expf and a division have two in thirty.  8192 x 2 x 12288 bf16, whose
// bytes take 78 us: 96; with the step 102, with expf and a division 166.
__device__ __forceinline__ float f8_silu_mul(float g, float u) {
    const float c = 1.44269502162933349609375f;                            // log2 e to f32
    const float h = fminf(fmaxf(g, -90.f), 88.f), t = h * -c, lo = fmaf(h, -c, -t);
    float z, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(z) : "f"(t - 2.f));
    z = fmaf(z, fmaf(h, -1.3349758e-8f, lo * 0.69314718f), z);             // (log2 e - c) ln 2 = 1.3349758e-8
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(0.25f + z));
    return g * (r * 0.25f) * u;
}

// values of an input row (its 2 K pass an int's range where K is the largest that is taken)
__host__ __device__ constexpr long long f8_row_values(bool gated, int K) { return (gated ? 2LL : 1LL) * K; }
static_assert(f8_row_values(true, 1 << 30) == 1LL << 31, "counted in 64 bits");

// A warp takes 512 columns of a row (four blocks) at a time and asks for U such pieces before it works on the first.
template <typename T, bool GATED, bool VEC, int U>
__global__ void __launch_bounds__(256)
f8_rows_kernel(const T* x, long long ldx, long long M, int K, F8Out o) {
    const int c0 = f8_col(threadIdx.x & 31), per = (K + 511) / 512;
    const unsigned warps = gridDim.x * 8, w = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int dm = (int)(warps / per), dc = (int)(warps % per);             // a step of all warps: rows and pieces
    long long m = w / per;
    int piece = (int)(w % per);
    const T* x_end = x + (M - 1) * ldx + f8_row_values(GATED, K);
    pdl_wait();
    pdl_launch_dependents();
    while (m < M) {
        F8Chunk<T, VEC> v[U][2], g[GATED ? U : 1][2];
        long long row[U];
        int col[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            row[u] = m; col[u] = piece * 512 + c0;
            const T* at = x + (m < M ? m : 0) * ldx;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = col[u] + 64 * h;
                const bool in = m < M && c < K;
                if constexpr (GATED) g[u][h].load(at, in ? c : 0, K, in, x, x_end);
                v[u][h].load(at + (GATED ? K : 0), in ? c : 0, K, in, x, x_end);
            }
            m += dm; piece += dc;
            if (piece >= per) { piece -= per; ++m; }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (row[u] >= M) break;                                          // (the warp as one)
            float y[2][8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                v[u][h].get(y[h], col[u] + 64 * h, K);
                if constexpr (GATED) {
                    float gate[8];
                    g[u][h].get(gate, col[u] + 64 * h, K);
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[h][i] = f8_silu_mul(gate[i], y[h][i]);
                }
            }
            f8_emit<VEC>(y, row[u], col[u], K, true, o);
        }
    }
}

struct F8NormArgs { F8Norm n; long long M; int K, tpr; bool vec_w; F8Out o; };
// `tpr` threads have a row (a block several, where it has fewer columns than 16 x 256), PER times 16 columns each, in registers between the sum and the codes; PER = 0: wider rows,
// read again for the codes (what the block stored ahead of the sum's barrier, where there is a residual).  A block keeps its weights in registers over the rows it takes in turn, and asks for the
// next row before it finishes one.
template <typename T, typename R, bool VEC, int PER>
__global__ void __launch_bounds__(512)
f8_norm_kernel(const F8NormArgs a) {
    constexpr bool RES = !std::is_same<R, void>::value;
    using RT = typename std::conditional<RES, R, T>::type;
    __shared__ float red[2][16];
    const int rpb = blockDim.x / a.tpr, sub = threadIdx.x / a.tpr, t = threadIdx.x - sub * a.tpr, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, K = a.K;
    const T* x = static_cast<const T*>(a.n.x);
    const RT* res = static_cast<const RT*>(a.n.residual);
    RT* res_out = static_cast<RT*>(a.n.residual_out);
    const T* x_end = x + (a.M - 1) * a.n.ldx + K;
    const long long r_len = (a.M - 1) * a.n.ldr + K;
    struct Piece { F8Chunk<T, VEC> x[2]; F8Chunk<RT, VEC> r[2]; };
    auto load = [&](long long m, int c0, Piece& p) {
        const long long at = m < a.M ? m : 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = c0 + 64 * h;
            const bool in = m < a.M && c < K;
            p.x[h].load(x + at * a.n.ldx, in ? c : 0, K, in, x, x_end);
            if constexpr (RES) p.r[h].load(res + at * a.n.ldr, in ? c : 0, K, in, res, res + r_len);
        }
    };
    auto sum = [&](long long m, int c0, const Piece& p, float (*v)[8]) {       // h of 16 columns, stored where there is a residual -> their squares
        const long long at = m < a.M ? m : 0;
        float s = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = c0 + 64 * h;
            p.x[h].get(v[h], c, K);
            if constexpr (RES) {
                float r[8];
                p.r[h].get(r, c, K);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[h][i] += r[i];
                f8_store8<RT, VEC>(res_out + at * a.n.ldr, c, K, m < a.M, v[h]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[h][i] * v[h][i];
        }
        return s;
    };
    auto row_rstd = [&](float s, int turn) {
        s = warp_sum(s);
        if (a.tpr > 32) {
            const int nw = a.tpr >> 5, w0 = sub * nw;
            if (lane == 0) red[turn & 1][warp] = s;
            __syncthreads();                        // (the other half of `red` is the next row's: nobody is still reading it)
            s = warp_sum(lane < nw ? red[turn & 1][w0 + lane] : 0.f);
        }
        return rsqrtf(s / (float)K + a.n.eps);
    };
    auto weights = [&](int c0, float (*w)[8]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (c0 + 64 * h < K) f8_load8(a.n.w, a.n.w_type, 0, c0 + 64 * h, K, a.vec_w, w[h]);
            else {
#pragma unroll
                for (int i = 0; i < 8; ++i) w[h][i] = 0.f;
            }
        }
    };
    const long long step = (long long)gridDim.x * rpb;
    long long base = (long long)blockIdx.x * rpb;
    const int c0 = f8_col(t);
    int turn = 0;
    pdl_wait();
    pdl_launch_dependents();
    if constexpr (PER > 0) {
        float w[PER][2][8];
        constexpr bool AHEAD = VEC || PER == 1 || !RES;       // (the pieces of 32 columns and a residual's would not stay in registers: 2048 x 9290 bf16 and f32 114 us so, 84 without; of 16 columns they do: 8192 x 4099 bf16 114, 124 without)
        Piece p[PER];
        if (AHEAD) {
#pragma unroll
            for (int j = 0; j < PER; ++j) load(base + sub, c0 + j * a.tpr * 16, p[j]);
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) weights(c0 + j * a.tpr * 16, w[j]);
        for (; base < a.M; base += step, ++turn) {
            const long long m = base + sub;
            float v[PER][2][8], s = 0.f;
            if (!AHEAD) {
#pragma unroll
                for (int j = 0; j < PER; ++j) load(m, c0 + j * a.tpr * 16, p[j]);
            }
#pragma unroll
            for (int j = 0; j < PER; ++j) s += sum(m, c0 + j * a.tpr * 16, p[j], v[j]);
            if (AHEAD && base + step < a.M) {
#pragma unroll
                for (int j = 0; j < PER; ++j) load(m + step, c0 + j * a.tpr * 16, p[j]);
            }
            const float rstd = row_rstd(s, turn);             // y = (x rstd) w in this order: x w may not have a place in f32 where y has
#pragma unroll
            for (int j = 0; j < PER; ++j) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[j][h][i] = v[j][h][i] * rstd * w[j][h][i];
                f8_emit<VEC>(v[j], m, c0 + j * a.tpr * 16, K, m < a.M, a.o);
            }
        }
    } else {
        for (; base < a.M; base += step, ++turn) {
            const long long m = base + sub;
            float s = 0.f;
            for (int i0 = 0; i0 < K; i0 += a.tpr * 16) {        // (all threads alike: shuffles)
                Piece p;
                float v[2][8];
                load(m, i0 + c0, p);
                s += sum(m, i0 + c0, p, v);
            }
            const float rstd = row_rstd(s, turn);
            for (int i0 = 0; i0 < K; i0 += a.tpr * 16) {
                const int c = i0 + c0;
                float v[2][8], w[2][8];
                weights(c, w);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const bool in = m < a.M && c + 64 * h < K;
                    if constexpr (RES) {
                        F8Chunk<RT, VEC> q;
                        q.load(static_cast<const RT*>(res_out) + (in ? m : 0) * a.n.ldr, in ? c + 64 * h : 0, K, in, res_out, res_out + r_len);
                        q.get(v[h], c + 64 * h, K);
                    } else {
                        F8Chunk<T, VEC> q;
                        q.load(x + (in ? m : 0) * a.n.ldx, in ? c + 64 * h : 0, K, in, x, x_end);
                        q.get(v[h], c + 64 * h, K);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[h][i] = in ? v[h][i] * rstd * w[h][i] : 0.f;
                }
                f8_emit<VEC>(v, m, c, K, m < a.M, a.o);
            }
        }
    }
}

static bool f8_aligned(const void* p, long long ld, int type) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * f8_bytes(type)) % 16 == 0; }
// blocks of a kernel that the current device runs at once
template <typename F>
static int f8_resident(F kernel, int threads, std::atomic<int>* known) {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= CB_MAX_DEV) return 148;
    n = known[dev].load(std::memory_order_relaxed);
    if (!n) {
        int sms = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
            cudaGetLastError();
            return 148;
        }
        n = n > 0 ? n * sms : sms;
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

template <typename T, bool GATED, bool VEC>
static int f8_rows_v(cudaStream_t st, const void* x, long long ldx, long long M, int K, const F8Out& out, bool pdl) {
    constexpr int U = VEC && !GATED ? 2 : 1;
    static std::atomic<int> known[CB_MAX_DEV];
    const long long pieces = M * ((K + 511) / 512);
    const long long blocks = std::min<long long>((pieces + 7) / 8, f8_resident(f8_rows_kernel<T, GATED, VEC, U>, 256, known));
    return launch_k(f8_rows_kernel<T, GATED, VEC, U>, dim3((unsigned)blocks), dim3(256), 0, st, pdl, static_cast<const T*>(x), ldx, M, K, out);
}
template <typename T, bool GATED>
static int f8_rows_t(cudaStream_t st, const void* x, int type, long long ldx, long long M, int K, const F8Out& out, bool pdl) {
    return f8_aligned(x, ldx, type) && K % 8 == 0 ? f8_rows_v<T, GATED, true>(st, x, ldx, M, K, out, pdl) : f8_rows_v<T, GATED, false>(st, x, ldx, M, K, out, pdl);
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

template <typename T, typename R, bool VEC, int PER>
static int f8_norm_p(cudaStream_t st, const F8NormArgs& a, int block, bool pdl) {
    static std::atomic<int> known[17][CB_MAX_DEV];              // by the block's warps
    const int rows = block / a.tpr;
    const long long blocks = std::min<long long>((a.M + rows - 1) / rows, f8_resident(f8_norm_kernel<T, R, VEC, PER>, block, known[block / 32]));
    return launch_k(f8_norm_kernel<T, R, VEC, PER>, dim3((unsigned)blocks), dim3(block), 0, st, pdl, a);
}
template <typename T, typename R, bool VEC>
static int f8_norm_v(cudaStream_t st, F8NormArgs& a, bool pdl) {
    // whole warps for a row, as few as have its columns (power of two: 8192 x 4099 bf16 and a residual 133 us, so 114); a block of about 256 threads
    a.tpr = std::min(512, (a.K + F8_BLOCK - 1) / F8_BLOCK * 8 + 31 & ~31);
    const int block = a.tpr * std::max(1, 256 / a.tpr);
    if (a.K <= a.tpr * 16) return f8_norm_p<T, R, VEC, 1>(st, a, block, pdl);
    if (a.K <= a.tpr * 32) return f8_norm_p<T, R, VEC, 2>(st, a, block, pdl);
    return f8_norm_p<T, R, VEC, 0>(st, a, block, pdl);
}
template <typename T, typename R>
static int f8_norm_r(cudaStream_t st, F8NormArgs& a, bool pdl) {
    const F8Norm& n = a.n;
    const bool vec = a.K % 8 == 0 && f8_aligned(n.x, n.ldx, n.type) && (!n.residual || (f8_aligned(n.residual, n.ldr, n.res_type) && f8_aligned(n.residual_out, n.ldr, n.res_type)));
    return vec ? f8_norm_v<T, R, true>(st, a, pdl) : f8_norm_v<T, R, false>(st, a, pdl);
}
template <typename T>
static int f8_norm_t(cudaStream_t st, F8NormArgs& a, bool pdl) {
    if (!a.n.residual) return f8_norm_r<T, void>(st, a, pdl);
    switch (a.n.res_type) {
        case F8_F32:  return f8_norm_r<T, float>(st, a, pdl);
        case F8_BF16: return f8_norm_r<T, bf16>(st, a, pdl);
        case F8_F16:  return f8_norm_r<T, __half>(st, a, pdl);
        default: return -1000;
    }
}
int f8_rms_norm_launch(cudaStream_t st, const F8Norm& n, long long M, int K, const F8Out& out, bool pdl) {
    if (M == 0) return 0;
    F8NormArgs a = {n, M, K, 0, f8_aligned(n.w, 0, n.w_type), out};
    switch (n.type) {
        case F8_F32:  return f8_norm_t<float>(st, a, pdl);
        case F8_BF16: return f8_norm_t<bf16>(st, a, pdl);
        case F8_F16:  return f8_norm_t<__half>(st, a, pdl);
        default: return -1000;
    }
}

}  // namespace cb
