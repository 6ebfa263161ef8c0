// A paged key/value cache in 8 bits (e4m3) with a scale for each page and head: rows into the cache (kv8_append.cu), attention over it (kv8_attention.cu).
//
// Codes of keys and of values lie [pages, kv heads, page, D], the two scales of a page and head side by side, [pages, kv heads, 2].  A value is code * scale.
#pragma once

#include "common.cuh"
#include "kv8_units.h"

namespace cb {

enum Kv8Type : int { KV8_F32 = 0, KV8_BF16 = 1, KV8_F16 = 2 };      // crane_b200_dtype

struct Kv8Rows { const void* p; int type; long long ld, ldh; };     // [rows, heads, D]: rows ld, heads ldh elements apart, columns side by side

int kv8_append_launch(cudaStream_t st, const Kv8Rows& k, const Kv8Rows& v, const Kv8Pool& pool, const Kv8Seqs& s, bool pdl);

struct Kv8Attention { Kv8Rows q; void* out; long long ldo, ldoh; int heads; float scale; int max_rows; void* work; int* err; };
size_t kv8_attention_bytes(int type, int heads, int kv_heads, int dim, int rows, int seqs, int max_rows);      // of `work`, on the current device
int kv8_attention_launch(cudaStream_t st, const Kv8Attention& a, const Kv8Pool& pool, const Kv8Seqs& s, bool pdl);

// Sequences with many rows of 16 bits, D up to 128 (kv8_flash.cu); kv8_attention_launch's business
constexpr int KV8_FLASH_ROWS = 256;
int kv8_flash_launch(cudaStream_t st, const Kv8Attention& a, const Kv8Deal& d, Kv8Join* joins, float* parts, bool pdl);

// `work` begins with a Kv8Join for each CTA, the parts follow
constexpr size_t kv8_joins(int ctas) { return (size_t)ctas * sizeof(Kv8Join); }

#ifdef __CUDACC__
// The steps of all sequences (kv8_units.h) and, in `sums`, those ahead of each of the KV8_SHARES equal shares of the sequences.  Every thread of the block.
constexpr int KV8_SHARES = 128;
template <typename U>
__device__ __forceinline__ long long kv8_count(const Kv8Deal& d, long long (&sums)[KV8_SHARES + 1]) {
    const int tid = threadIdx.x, per = (d.s.seqs + KV8_SHARES - 1) / KV8_SHARES;
    long long mine = 0;
    if (tid < KV8_SHARES)
        for (int i = tid * per; i < min(d.s.seqs, tid * per + per); ++i) {
            U u;
            u.b = i;
            u.shape(d);
            mine += u.head_steps(d) * d.p.kv_heads;
        }
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const long long t = __shfl_up_sync(0xffffffffu, incl, o); if ((tid & 31) >= o) incl += t; }
    __shared__ long long wsum[KV8_SHARES / 32];
    if ((tid & 31) == 31 && tid < KV8_SHARES) wsum[tid >> 5] = incl;
    __syncthreads();
    long long before = 0, all = 0;
    for (int w = 0; w < KV8_SHARES / 32; ++w) { if (w < (tid >> 5)) before += wsum[w]; all += wsum[w]; }
    if (tid < KV8_SHARES) sums[tid] = before + incl - mine;
    if (tid == 0) sums[KV8_SHARES] = all;
    __syncthreads();
    return all;
}
template <typename U>
__device__ __forceinline__ U kv8_find(const Kv8Deal& d, const long long (&sums)[KV8_SHARES + 1], long long step) {
    int lo = 0, n = KV8_SHARES;                // the last share that begins at or ahead of the step
    while (n > 1) { const int h = n / 2; if (sums[lo + h] <= step) { lo += h; n -= h; } else n = h; }
    U u;
    u.seek(d, lo * ((d.s.seqs + KV8_SHARES - 1) / KV8_SHARES), sums[lo], step);
    return u;
}
#endif

}  // namespace cb
