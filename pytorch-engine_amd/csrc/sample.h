// Token sampling (sample.hip): what the entry point hands over, validated.
#pragma once

#include "common.h"

namespace pgmoe {

constexpr int kMaxVocab = 1 << 20;

struct SampleArgs {
    const void* logits;
    int dtype;
    int64_t row_stride;
    int rows, vocab;
    const float* u;
    pgmoe_sampling P;
    int64_t* token;
    float* logprob;
    int shift;  // weights are held as multiples of 2^-shift
    void* ws;
};
size_t sample_ws_bytes(int rows, int vocab);
int launch_sample(const SampleArgs& A, hipStream_t st);

}  // namespace pgmoe
