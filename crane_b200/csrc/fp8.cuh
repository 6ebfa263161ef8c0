// Linears in 8-bit floating point (e4m3) with a scale for each block of 128: activation rows to codes (fp8_rows.cu), codes x codes^T (fp8_gemm.cu).
//
// A row's codes lie `ld` bytes apart, every row on a 16-byte boundary (TMA); its scales, one per 128 columns, are stored block by block: the scale of row m and
// block b at scales[b * lds + m], so that neighbouring rows' are neighbours.  Weights have a scale for each 128 x 128, [ceil(N / 128), ceil(K / 128)].
#pragma once

#include "common.cuh"

namespace cb {

constexpr int F8_BLOCK = 128;
constexpr int f8_blocks(long long n) { return (int)((n + F8_BLOCK - 1) / F8_BLOCK); }

enum F8Type : int { F8_F32 = 0, F8_BF16 = 1, F8_F16 = 2 };      // crane_b200_dtype
constexpr int f8_bytes(int t) { return t == F8_F32 ? 4 : 2; }

struct F8Out { unsigned char* codes; long long ld; float* scales; long long lds; };
struct F8Rows { const unsigned char* codes; long long ld; const float* scales; long long lds; };

// rows as they are; [gate | up] rows of 2 K columns -> SiLU(gate) * up
int f8_quantize_launch(cudaStream_t st, const void* x, int type, long long ldx, long long M, int K, const F8Out& out, bool pdl);
int f8_silu_mul_launch(cudaStream_t st, const void* x, int type, long long ldx, long long M, int K, const F8Out& out, bool pdl);
// h = x + residual, rounded to the residual's type and stored to residual_out (may be `residual`); codes of h * rsqrt(mean h^2 + eps) * w
struct F8Norm {
    const void* x; int type; long long ldx;
    const void* residual; void* residual_out; int res_type; long long ldr;     // residual == nullptr: h = x
    const void* w; int w_type; float eps;
};
int f8_rms_norm_launch(cudaStream_t st, const F8Norm& a, long long M, int K, const F8Out& out, bool pdl);

// out[m, n] = add[m, n] + sum_b x.scales[b, m] ws[n / 128, b] sum_{k in b} x[m, k] w[n, k];  `add` has out's type, rows ldadd apart, and may be `out`
struct F8Linear {
    F8Rows x;
    const unsigned char* w; long long ldw; const float* ws; long long ldws;
    void* out; int type; long long ldo;
    const void* add; long long ldadd;
    bool w_static;             // no kernel that may still run writes the weights: their first tiles are fetched ahead of the dependency wait
    int* err = nullptr;        // word of bounded waits that run out (TcWait); nullptr: the stream's, which calls that read results from that stream look at
};
int f8_linear_launch(cudaStream_t st, const F8Linear& a, int M, int N, int K, bool pdl);

// The stream's error word (TcWait) without disturbing a capture that is under way on this thread
int f8_err_word(cudaStream_t st, int** out);

}  // namespace cb
