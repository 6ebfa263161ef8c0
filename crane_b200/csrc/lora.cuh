// Low-rank adapters of many requests beside a shared projection: out_i = add_i + scale_w B_w (A_w x_i) with w = which_i (lora.cu).
#pragma once

#include "common.cuh"

namespace cb {

enum LoraType : int { LORA_F32 = 0, LORA_BF16 = 1, LORA_F16 = 2 };   // crane_b200_dtype

struct Lora {
    const void* x; int type; long long ldx;                         // [m, k]; add and out have its type
    const void* a; const void* b; int w_type;                       // [adapters, rank, k], [adapters, n, rank], contiguous; w_type = type, or any beside f32 rows
    const int* which;                                               // [m]; outside [0, adapters): none
    const float* scales;                                            // [adapters]; nullptr: ones
    const void* add; long long ldadd;                               // nullptr: zeros; may be out
    void* out; long long ldo;
    int m, n, k, rank, adapters;
    int* err;                                                       // tc_err_word, or the like: of a wait that ran out
};
constexpr int LORA_MAX_RANK = 128;
// Many rows of 16 bits, ranks from 17 to 64, everything on 16-byte boundaries (lora_tiles.cu)
int lora_tiles_launch(cudaStream_t st, const Lora& l, bool pdl);
int lora_linear_launch(cudaStream_t st, const Lora& l, bool pdl);

}  // namespace cb
