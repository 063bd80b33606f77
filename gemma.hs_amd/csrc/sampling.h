// Batched sampling with top-k, top-p and min-p: launcher.
#pragma once

#include "common.h"

namespace gh {

// Up to SMP_BATCH rows in the order in which their workgroups start, by value
// in a kernel's arguments: each one's rules, and which of the call's it is.
constexpr int SMP_BATCH = 128;
struct SmpRule : gh_sampling {
    int row;
};
struct SmpRules {
    SmpRule r[SMP_BATCH];
};

constexpr int SMP_MAX_VOCAB = 1 << 24;
// Weights are integers: 2^smp_bits(n) for the largest logit, so that the sum
// of n of them fits into 63 bits.
inline int smp_bits(int n) {
    int b = 0;
    while ((int64_t(1) << b) < n) ++b;
    return std::min(51, 62 - b);
}

// Steps between a row's largest and smallest logit, elements that the exact
// search sorts, workgroups a row and groups a row at most.  Of 2048 steps one
// holds some 600 of 262144 normal logits, a list of 4096 leaves room for ties
// and for three searches at once (64 rows of mixed rules 70 us; by 1024 steps
// 81).
constexpr int SMP_BINS = 2048, SMP_LIST = 4096, SMP_CHUNKS = 64, SMP_GROUPS = 1024;

// What the bins alone say of a row's searches.
struct SmpCuts {
    unsigned long long total;   // mass of all
    unsigned long long upto_m;  // min_p: mass of the bins that it cannot reach behind
    int lo[4], hi[4];           // bins whose elements decide: top_k, top_p, min_p, the draw (lo > hi: none)
    int k, p, m;                // which of the rules cut anything off
};

// Device scratch of a row that several workgroups read.
struct SmpRow {
    unsigned long long mass[SMP_BINS], run_mass[SMP_BINS], list[SMP_LIST], first[SMP_CHUNKS];
    unsigned count[SMP_BINS], run_count[SMP_BINS];
    float low[SMP_CHUNKS];
    unsigned nan[SMP_CHUNKS];
    float group_max[SMP_GROUPS];  // largest logit of each group
    SmpCuts cuts;
    unsigned n_list;
    int is_short;  // 0: long; 1: the list has all the mass that counts; 2: mass[0] has the row's
};

// Workgroups a row; 0: one, which runs every step in one launch (no scratch).
// It saves three launches, and reads the row three times alone: 8 rows of
// 16384 logits take 30 us so and 36 by chunks, a single one of 32000 37 and 31
// (top-k 26 and 29), 64 of 32000 38 and 40.  Each chunk clears, fills and adds
// up bins of its own: 4096 logits for a few rows (one of 262144 33.2 us, by
// 8192 33.9), 8192 for more (16 rows 43, by 4096 49, by 16384 44).
inline int smp_chunks(int n_rows, int vocab) {
    if (vocab <= (n_rows <= 4 ? 20000 : 32768)) return 0;
    const int least = n_rows <= 4 ? 4096 : 8192;  // logits a workgroup
    return std::max(1, std::min({SMP_CHUNKS, 1024 / n_rows, (vocab + least - 1) / least}));
}

int launch_sample_rows(const float* logits, int n_rows, int vocab, const SmpRules& rules, SmpRow* scratch, int32_t* tokens,
                       hipStream_t s);

}  // namespace gh
