// Host side of the batched sampler: the checks of its rules.
#include <algorithm>
#include <cmath>

#include "host.h"
#include "sampling.h"

using namespace gh;

namespace {

// How much work a row is likely to be: weights of the whole row, a list of its
// first elements, its largest one.
int work_of(const gh_sampling& r) {
    if (r.temperature == 0.0f) return 0;
    return r.top_k == 0 || r.top_k > SMP_GROUPS / 4 ? 2 : 1;
}

}  // namespace

extern "C" int gh_sample_rows(gh_ctx* ctx, const float* logits, int32_t n_rows, int32_t vocab, const gh_sampling* rules,
                              int32_t* tokens_out) {
    OP_ENTER(ctx);
    if (n_rows < 0 || vocab <= 0 || vocab > SMP_MAX_VOCAB)
        return set_error(GH_ERR_INVALID, "gh_sample_rows: %d rows of %d logits", n_rows, vocab);
    if (n_rows == 0) return GH_OK;
    if (!logits || !rules || !tokens_out) return set_error(GH_ERR_INVALID, "gh_sample_rows: null argument");
    if (((uintptr_t)logits | (uintptr_t)tokens_out) & 3)
        return set_error(GH_ERR_INVALID, "gh_sample_rows: logits and tokens_out must be 4-byte aligned device pointers");
    for (int i = 0; i < n_rows; ++i) {
        const gh_sampling& r = rules[i];
        if (!(r.temperature >= 0.0f) || std::isinf(r.temperature))
            return set_error(GH_ERR_RANGE, "gh_sample_rows: row %d: temperature must be finite and >= 0", i);
        if (r.top_k < 0) return set_error(GH_ERR_RANGE, "gh_sample_rows: row %d: top_k %d", i, r.top_k);
        if (!(r.top_p >= 0.0f && r.top_p <= 1.0f) || !(r.min_p >= 0.0f && r.min_p <= 1.0f))
            return set_error(GH_ERR_RANGE, "gh_sample_rows: row %d: top_p %g or min_p %g outside [0, 1]", i, r.top_p, r.min_p);
        if (!(r.u >= 0.0f && r.u < 1.0f)) return set_error(GH_ERR_RANGE, "gh_sample_rows: row %d: u %g outside [0, 1)", i, r.u);
    }
    void* scratch = nullptr;
    if (smp_chunks(1, vocab)) GH_CHECK(ctx_scratch(ctx, sizeof(SmpRow) * std::min(n_rows, SMP_BATCH), &scratch));
    for (int i = 0; i < n_rows; i += SMP_BATCH) {
        SmpRules b;
        const int m = std::min(n_rows - i, SMP_BATCH);
        // Rows of like work one behind the other, so that each CU gets some of
        // every kind: in the caller's order those with the same rules may meet
        // on the same CUs (64 rows whose rules repeat: 86 us
        // so, 76 in this).
        int at = 0;
        for (int work = 2; work >= 0; --work)
            for (int j = 0; j < m; ++j)
                if (work_of(rules[i + j]) == work) b.r[at++] = {rules[i + j], j};
        GH_CHECK(launch_sample_rows(logits + (size_t)i * vocab, m, vocab, b, (SmpRow*)scratch, tokens_out + i, ctx->stream));
    }
    return op_sync(ctx);
}
