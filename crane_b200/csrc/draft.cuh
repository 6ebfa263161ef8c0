// Verification of drafted tokens against the target's probabilities, from given random numbers (draft.cu).
#pragma once

#include "common.cuh"

namespace cb {

enum DraftType : int { DRAFT_F32 = 0, DRAFT_BF16 = 1, DRAFT_F16 = 2 };      // crane_b200_dtype

struct Draft {
    const void* logits; int type; long long ld;        // [total + seqs, vocab]: sequence b's rows are starts[b] + b .. starts[b + 1] + b
    const void* q; long long ldq;                      // the draft model's [total, vocab], of the same type; nullptr: each draft was certain
    const int* tokens; const int* starts;              // [total], [seqs + 1]
    const float* temperatures;                         // [seqs]; nullptr: 1
    const float* uniforms; const float* noise; long long ldn;      // [total], [seqs, vocab]
    int vocab, seqs, total;
    int* accepted; int* next;                          // [seqs]
    void* work;
};
size_t draft_bytes(int seqs, int total, int vocab, bool q);         // of `work`, on the current device
int draft_verify_launch(cudaStream_t st, const Draft& d, bool pdl);

}  // namespace cb
