// The choice of a token for each row of logits, from given random numbers.
#pragma once

#include "common.hpp"

namespace th {

// Sums of weights are 64-bit integers; a row of 2^20 leaves each weight 42 bits.
constexpr size_t SAMPLE_MAX_VOCAB = (size_t)1 << 20;

struct SampleArgs {
    const void* x;  // [rows][vocab]
    th_dtype xdt;
    const float *u, *temp, *top_p, *min_p;  // [rows]; all but u may be null
    const uint32_t* top_k;
    uint32_t* token;
    float* prob;  // or null
    int rows, vocab;
};
void launch_sample_rows(const SampleArgs& a, hipStream_t s);

}  // namespace th
