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
size_t kv8_attention_bytes(int heads, int kv_heads, int dim, int rows, int seqs, int max_rows);      // of `work`, on the current device
int kv8_attention_launch(cudaStream_t st, const Kv8Attention& a, const Kv8Pool& pool, const Kv8Seqs& s, bool pdl);

}  // namespace cb
