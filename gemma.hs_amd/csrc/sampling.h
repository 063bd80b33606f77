// Batched sampling with top-k, top-p and min-p: launcher.
#pragma once

#include "common.h"

namespace gh {

// Rules of up to SMP_BATCH rows, by value in a kernel's arguments.
constexpr int SMP_BATCH = 128;
struct SmpRules {
    gh_sampling r[SMP_BATCH];
};

constexpr int SMP_MAX_VOCAB = 1 << 24;
// Weights are integers: 2^smp_bits(n) for the largest logit, so that the sum
// of n of them fits into 63 bits.
inline int smp_bits(int n) {
    int b = 0;
    while ((int64_t(1) << b) < n) ++b;
    return std::min(52, 62 - b);
}

int launch_sample_rows(const float* logits, int n_rows, int vocab, const SmpRules& rules, int32_t* tokens, hipStream_t s);

}  // namespace gh
