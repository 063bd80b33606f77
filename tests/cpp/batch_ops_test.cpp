// The host side of the batched operators (gh_kv8_*, gh_sample_rows) on the
// CPU: every refusal with its code, what a call hands to the kernels, lengths,
// and lifetimes.  Linked against hip_stub.cpp / kernel_stub.cpp and the
// launchers below, which check each launch against the cache's shape instead
// of running it; built with AddressSanitizer by tests/test_batch_ops_host.py.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <limits>
#include <numeric>
#include <thread>
#include <vector>

#include "../../gemma.hs_amd/csrc/kv8.h"
#include "../../gemma.hs_amd/csrc/sampling.h"

extern "C" size_t hip_stub_live_bytes(void);
extern "C" void hip_stub_set_device_bytes(size_t n);

#define CHECK(c)                                                                                                        \
    do {                                                                                                                \
        if (!(c)) {                                                                                                     \
            std::fprintf(stderr, "FAIL %s:%d: %s (last error: %s)\n", __FILE__, __LINE__, #c, gh_last_error());         \
            return 1;                                                                                                   \
        }                                                                                                               \
    } while (0)

// ---- launchers that look at their arguments
namespace gh {
int bad_launches = 0, launches = 0;
int cap_tokens = 0;  // nb * 64 of the cache under test
int n_seq = 0;
std::vector<Kv8Batch> batches;
std::vector<Att8> attentions;
std::vector<int> sample_rows;
std::vector<char> covered;        // of a call's tokens: once each, in whichever launch
const float* rows_at = nullptr;  // first row of the calls, where tokens are watched
#define WANT(c)                                                             \
    do {                                                                    \
        if (!(c)) {                                                         \
            ++bad_launches;                                                 \
            std::fprintf(stderr, "bad launch %s:%d: %s\n", __FILE__, __LINE__, #c); \
        }                                                                   \
    } while (0)
static void look(const Kv8Batch& b, int n) {
    ++launches;
    WANT(n > 0 && n <= KV8_BATCH);
    for (int i = 0; i < n; ++i) WANT(b.seq[i] >= 0 && b.seq[i] < n_seq && b.pos[i] >= 0);
    batches.push_back(b);
}
static void cover(const Kv8Batch& b, int n, const float* rows, size_t ld) {
    const size_t first = rows_at ? (rows - rows_at) / ld : 0;
    for (int i = 0; rows_at && i < n; ++i)
        for (size_t t = first + b.off[i]; t < first + b.off[i] + b.cnt[i]; ++t) {
            if (t >= covered.size()) covered.resize(t + 1, 0);
            WANT(!covered[t]);
            covered[t] = 1;
        }
}
int launch_kv8_append(const Kv8Dev& c, int hd, const Kv8Batch& b, int n, int blocks, const float* k, const float* v, hipStream_t) {
    look(b, n);
    WANT(k && v);
    cover(b, n, k, (size_t)c.nkv * hd);
    int most = 0;
    for (int i = 0; i < n; ++i) {
        const int cnt = b.cnt[i], end = b.pos[i] + cnt;
        WANT(cnt > 0 && end <= cap_tokens);
        most = std::max(most, (end - 1) / 64 - b.pos[i] / 64 + 1);
    }
    WANT(blocks == most && blocks > 0);
    return GH_OK;
}
int launch_kv8_truncate(const Kv8Dev&, int, const Kv8Batch& b, int n, hipStream_t) {
    look(b, n);
    for (int i = 0; i < n; ++i) WANT(b.cnt[i] % 64 != 0 && b.cnt[i] < b.pos[i]);
    return GH_OK;
}
int launch_kv8_read(const Kv8Dev&, int, const Kv8Batch& b, int n, int blocks, float* k, float* v, hipStream_t) {
    look(b, n);
    WANT((k || v) && blocks > 0);
    for (int i = 0; i < n; ++i) WANT(b.cnt[i] >= 0 && b.pos[i] + b.cnt[i] <= cap_tokens);
    return GH_OK;
}
int launch_kv8_attention(const Kv8Dev& c, int hd, const Kv8Batch& b, int n, const Att8& a, hipStream_t) {
    look(b, n);
    attentions.push_back(a);
    WANT(a.q && a.out && a.group * c.nkv == a.heads && (a.tile == 4 || a.tile == 16) && a.tiles > 0 && a.ns > 0);
    cover(b, n, a.q, (size_t)a.heads * hd);
    int part = 0, most_q = 0;  // every query token has its own place among the states
    for (int i = 0; i < n; ++i) {
        WANT(b.part[i] == part && b.cnt[i] > 0);
        part += b.cnt[i];
        most_q = std::max(most_q, b.cnt[i]);
    }
    WANT((size_t)part * a.heads == a.rows && most_q == a.most_q);
    WANT((int64_t)a.ns * a.tiles * c.nkv < 1 << 24);
    if (a.tile == 4) WANT(a.tiles == 1);
    if (a.ns > 1) {  // the scratch holds every state
        WANT(a.part != nullptr);
        if (a.part) std::memset(a.part, 0, a.rows * a.ns * (hd + 2) * sizeof(float));
    }
    for (int i = 0; i < n; ++i) {
        const int rows = b.cnt[i] * a.group;
        WANT(rows <= a.tiles * a.tile && b.pos[i] <= cap_tokens);
        for (int r : {0, 1, rows / 2, rows - 1})
            if (r >= 0 && a.group > 1) WANT((int)(((uint64_t)r * a.group_inv) >> 32) == r / a.group);
        // the chunks cover every tile's blocks
        for (int row0 = 0; row0 < rows; row0 += a.tile) {
            const int last = std::min(rows, row0 + a.tile) - 1, n_q = rows / a.group;
            const int p0 = b.pos[i] - n_q + row0 / a.group, p1 = b.pos[i] - n_q + last / a.group;
            const int begin = a.window ? std::max(p0 - a.window + 1, 0) / 64 : 0, end = p1 < 0 ? 0 : p1 / 64 + 1;
            WANT((int64_t)a.ns * a.chunk >= end - begin);
        }
    }
    return GH_OK;
}
int launch_sample_rows(const float* l, int n_rows, int vocab, const SmpRules&, SmpRow* scratch, int32_t* t, hipStream_t) {
    ++launches;
    WANT(l && t && n_rows > 0 && n_rows <= SMP_BATCH);
    const int chunks = smp_chunks(n_rows, vocab);
    WANT(chunks <= SMP_CHUNKS && (chunks > 0 || vocab <= 32768));
    if (chunks) {
        WANT(scratch != nullptr);
        if (scratch) std::memset(scratch, 0, sizeof(SmpRow) * n_rows);
    }
    sample_rows.push_back(n_rows);
    return GH_OK;
}
}  // namespace gh
using namespace gh;

namespace {

alignas(16) float buf[64];
float* const P = buf;

int cache(gh_ctx* ctx, int seqs, int max_seq, int nkv, int hd, gh_kv8** kv) {
    n_seq = seqs;
    cap_tokens = (max_seq + 63) / 64 * 64;
    return gh_kv8_create(ctx, seqs, max_seq, nkv, hd, kv);
}

int length(gh_kv8* kv, int s) {
    int32_t n = -1;
    return gh_kv8_length(kv, s, &n) == GH_OK ? n : -1;
}

int refusals() {
    gh_ctx* ctx = nullptr;
    CHECK(gh_ctx_create(0, &ctx) == GH_OK);
    gh_kv8* kv = nullptr;
    CHECK(gh_kv8_create(nullptr, 1, 64, 1, 64, &kv) == GH_ERR_INVALID);
    CHECK(gh_kv8_create(ctx, 1, 64, 1, 64, nullptr) == GH_ERR_INVALID);
    for (int bad : {0, -1}) {
        CHECK(gh_kv8_create(ctx, bad, 64, 1, 64, &kv) == GH_ERR_INVALID);
        CHECK(gh_kv8_create(ctx, 1, bad, 1, 64, &kv) == GH_ERR_INVALID);
        CHECK(gh_kv8_create(ctx, 1, 64, bad, 64, &kv) == GH_ERR_INVALID);
    }
    for (int hd : {0, 16, 48, 96, 512, -64}) CHECK(gh_kv8_create(ctx, 1, 64, 1, hd, &kv) == GH_ERR_INVALID);
    CHECK(gh_kv8_create(ctx, 1, (1 << 22) + 1, 1, 64, &kv) == GH_ERR_INVALID);
    hip_stub_set_device_bytes(1 << 20);
    CHECK(gh_kv8_create(ctx, 64, 4096, 8, 256, &kv) == GH_ERR_OOM);
    hip_stub_set_device_bytes(SIZE_MAX);
    CHECK(cache(ctx, 3, 100, 2, 64, &kv) == GH_OK);

    const int32_t s01[] = {0, 1}, s00[] = {1, 1}, s3[] = {3}, sm[] = {-1}, one[] = {1, 1}, neg[] = {-1}, zero[] = {0, 0};
    const int32_t h100[] = {100, 100}, h101[] = {101};
    // arrays
    CHECK(gh_kv8_append(kv, -1, s01, one, P, P) == GH_ERR_INVALID);
    CHECK(gh_kv8_append(kv, 1, nullptr, one, P, P) == GH_ERR_INVALID);
    CHECK(gh_kv8_append(kv, 1, s01, nullptr, P, P) == GH_ERR_INVALID);
    CHECK(gh_kv8_append(kv, 1, s3, one, P, P) == GH_ERR_INVALID);
    CHECK(gh_kv8_append(kv, 1, sm, one, P, P) == GH_ERR_INVALID);
    CHECK(gh_kv8_append(kv, 2, s00, one, P, P) == GH_ERR_INVALID);  // twice
    CHECK(gh_kv8_append(kv, 1, s01, neg, P, P) == GH_ERR_INVALID);
    CHECK(gh_kv8_append(kv, 1, s01, one, nullptr, P) == GH_ERR_INVALID);
    CHECK(gh_kv8_append(kv, 1, s01, one, P, nullptr) == GH_ERR_INVALID);
    CHECK(gh_kv8_append(kv, 1, s01, one, P + 1, P) == GH_ERR_INVALID);  // alignment
    CHECK(gh_kv8_append(kv, 1, s01, one, P, P + 3) == GH_ERR_INVALID);
    CHECK(gh_kv8_append(kv, 1, s01, h101, P, P) == GH_ERR_RANGE);
    CHECK(launches == 0 && length(kv, 0) == 0 && length(kv, 1) == 0);
    // nothing to do is no error
    CHECK(gh_kv8_append(kv, 0, nullptr, nullptr, nullptr, nullptr) == GH_OK);
    CHECK(gh_kv8_append(kv, 2, s01, zero, nullptr, nullptr) == GH_OK && launches == 0);
    CHECK(gh_kv8_append(kv, 2, s01, h100, P, P) == GH_OK && launches == 1);
    CHECK(length(kv, 0) == 100 && length(kv, 1) == 100 && length(kv, 2) == 0);
    // one entry too long: the others stay as they are
    const int32_t s21[] = {2, 1};
    CHECK(gh_kv8_append(kv, 2, s21, one, P, P) == GH_ERR_RANGE && length(kv, 2) == 0);
    int32_t n = 0;
    CHECK(gh_kv8_length(kv, 3, &n) == GH_ERR_INVALID && gh_kv8_length(kv, -1, &n) == GH_ERR_INVALID);
    CHECK(gh_kv8_length(kv, 0, nullptr) == GH_ERR_INVALID);

    // truncate
    CHECK(gh_kv8_truncate(kv, 1, s01, h101) == GH_ERR_RANGE);
    CHECK(gh_kv8_truncate(kv, 1, s01, neg) == GH_ERR_RANGE);
    CHECK(gh_kv8_truncate(kv, 2, s00, one) == GH_ERR_INVALID);
    CHECK(gh_kv8_truncate(kv, 1, s3, one) == GH_ERR_INVALID);
    CHECK(gh_kv8_truncate(kv, 1, s01, nullptr) == GH_ERR_INVALID);
    const int before = launches;
    const int32_t to[] = {64, 100};
    CHECK(gh_kv8_truncate(kv, 2, s01, to) == GH_OK && launches == before);  // a boundary and no change: no kernel
    CHECK(length(kv, 0) == 64 && length(kv, 1) == 100);
    const int32_t to2[] = {63, 70};
    CHECK(gh_kv8_truncate(kv, 2, s01, to2) == GH_OK && launches == before + 1);
    CHECK(batches.back().pos[0] == 64 && batches.back().cnt[0] == 63 && batches.back().pos[1] == 100);

    // read
    const int32_t b0[] = {0}, e63[] = {63}, e64[] = {64}, b9[] = {9}, e8[] = {8};
    CHECK(gh_kv8_read(kv, 1, s01, b0, e64, P, P) == GH_ERR_RANGE);
    CHECK(gh_kv8_read(kv, 1, s01, b9, e8, P, P) == GH_ERR_RANGE);
    CHECK(gh_kv8_read(kv, 1, s01, neg, e8, P, P) == GH_ERR_RANGE);
    CHECK(gh_kv8_read(kv, 1, s01, b0, e63, P + 2, P) == GH_ERR_INVALID);
    CHECK(gh_kv8_read(kv, 1, s01, nullptr, e63, P, P) == GH_ERR_INVALID);
    CHECK(gh_kv8_read(kv, 1, s01, b0, e63, nullptr, nullptr) == GH_OK && gh_kv8_read(kv, 1, s01, b9, b9, P, P) == GH_OK);
    CHECK(launches == before + 1);
    CHECK(gh_kv8_read(kv, 1, s01, b0, e63, P, nullptr) == GH_OK && launches == before + 2);

    // attention
    CHECK(gh_kv8_attention(kv, 1, s01, one, P, 3, 0, P) == GH_ERR_INVALID);  // heads
    CHECK(gh_kv8_attention(kv, 1, s01, one, P, 0, 0, P) == GH_ERR_INVALID);
    CHECK(gh_kv8_attention(kv, 1, s01, one, P, -2, 0, P) == GH_ERR_INVALID);
    CHECK(gh_kv8_attention(kv, 1, s01, one, P, 4, -1, P) == GH_ERR_INVALID);  // window
    CHECK(gh_kv8_attention(kv, 1, s01, neg, P, 4, 0, P) == GH_ERR_INVALID);
    CHECK(gh_kv8_attention(kv, 1, s3, one, P, 4, 0, P) == GH_ERR_INVALID);
    CHECK(gh_kv8_attention(kv, 1, s01, one, nullptr, 4, 0, P) == GH_ERR_INVALID);
    CHECK(gh_kv8_attention(kv, 1, s01, one, P, 4, 0, P + 1) == GH_ERR_INVALID);
    const int32_t many[] = {1 << 20};
    CHECK(gh_kv8_attention(kv, 1, s01, many, P, 4, 0, P) == GH_ERR_RANGE);
    CHECK(gh_kv8_attention(kv, 1, s01, one, P, 2 * 1025, 0, P) == GH_ERR_RANGE);
    CHECK(launches == before + 2);
    CHECK(gh_kv8_attention(kv, 1, s01, zero, nullptr, 4, 0, nullptr) == GH_OK && launches == before + 2);
    CHECK(gh_kv8_attention(kv, 2, s00, one, P, 4, 0, P) == GH_OK && launches == before + 3);  // the same sequence twice
    CHECK(gh_kv8_destroy(kv) == GH_OK);
    CHECK(gh_kv8_destroy(kv) == GH_ERR_STATE && gh_kv8_append(kv, 1, s01, one, P, P) == GH_ERR_STATE);
    CHECK(gh_kv8_length(nullptr, 0, &n) == GH_ERR_INVALID && gh_kv8_destroy(nullptr) == GH_OK);

    // sampler
    gh_sampling r[300];
    for (auto& x : r) x = {0.8f, 40, 0.9f, 0.1f, 0.5f};
    int32_t t[4];
    const int l0 = launches;
    CHECK(gh_sample_rows(nullptr, P, 1, 10, r, t) == GH_ERR_INVALID);
    CHECK(gh_sample_rows(ctx, nullptr, 1, 10, r, t) == GH_ERR_INVALID);
    CHECK(gh_sample_rows(ctx, P, 1, 10, nullptr, t) == GH_ERR_INVALID);
    CHECK(gh_sample_rows(ctx, P, 1, 10, r, nullptr) == GH_ERR_INVALID);
    CHECK(gh_sample_rows(ctx, P, -1, 10, r, t) == GH_ERR_INVALID);
    CHECK(gh_sample_rows(ctx, (float*)((char*)P + 2), 1, 10, r, t) == GH_ERR_INVALID);
    CHECK(gh_sample_rows(ctx, P, 1, 10, r, (int32_t*)((char*)t + 1)) == GH_ERR_INVALID);
    CHECK(gh_sample_rows(ctx, P, 1, 0, r, t) == GH_ERR_INVALID);
    CHECK(gh_sample_rows(ctx, P, 1, (1 << 24) + 1, r, t) == GH_ERR_INVALID);
    CHECK(gh_sample_rows(ctx, nullptr, 0, 10, nullptr, nullptr) == GH_OK);
    const float nan = std::nanf(""), inf = std::numeric_limits<float>::infinity();
    auto refused = [&](gh_sampling x) {
        r[2] = x;
        const int rc = gh_sample_rows(ctx, P, 3, 10, r, t);
        r[2] = r[0];
        return rc == GH_ERR_RANGE;
    };
    for (float x : {-0.1f, nan, inf}) CHECK(refused({x, 0, 1, 0, 0}));
    CHECK(refused({1, -1, 1, 0, 0}));
    for (float x : {-0.1f, 1.1f, nan, inf}) CHECK(refused({1, 0, x, 0, 0}) && refused({1, 0, 1, x, 0}) && refused({1, 0, 1, 0, x}));
    CHECK(refused({1, 0, 1, 0, 1.0f}));
    CHECK(launches == l0);
    CHECK(gh_sample_rows(ctx, P, 300, 10, r, t) == GH_OK && launches == l0 + 3 && sample_rows.back() == 300 - 2 * SMP_BATCH);
    CHECK(gh_sample_rows(ctx, P, 300, 262144, r, t) == GH_OK && launches == l0 + 6);
    CHECK(gh_ctx_destroy(ctx) == GH_OK);
    CHECK(bad_launches == 0 && hip_stub_live_bytes() == 0);
    return 0;
}

// What the attention hands to its kernels, over many shapes.
int splits() {
    gh_ctx* ctx = nullptr;
    rows_at = P;
    CHECK(gh_ctx_create(0, &ctx) == GH_OK);
    for (int nkv : {1, 2, 4}) {
        for (int max_seq : {1, 64, 700, 5000, 40000}) {
            gh_kv8* kv = nullptr;
            CHECK(cache(ctx, 300, max_seq, nkv, 32, &kv) == GH_OK);
            std::vector<int32_t> seqs(300), lens(300), nq(300);
            for (int i = 0; i < 300; ++i) {
                seqs[i] = 299 - i;
                lens[i] = (int)((int64_t)i * i * 7 % (max_seq + 1));
            }
            auto all = [](const std::vector<int32_t>& cnt, int n) {  // the call's tokens, each in one launch
                const size_t want = std::accumulate(cnt.begin(), cnt.begin() + n, (size_t)0);
                const bool ok = covered.size() == want && std::count(covered.begin(), covered.end(), 1) == (ptrdiff_t)want;
                covered.clear();
                return ok;
            };
            covered.clear();
            CHECK(gh_kv8_append(kv, 300, seqs.data(), lens.data(), P, P) == GH_OK && all(lens, 300));
            for (int group : {1, 2, 3, 4, 8, 20})
                for (int window : {0, 1, 512})
                    for (int t : {1, 2, 5, 33, 700}) {
                        for (int n : {1, 7, 300}) {
                            for (int i = 0; i < n; ++i) nq[i] = i % 3 == 2 ? 0 : std::max(0, t - i % 5);
                            CHECK(gh_kv8_attention(kv, n, seqs.data(), nq.data(), P, group * nkv, window, P) == GH_OK);
                            CHECK(all(nq, n));
                        }
                        // one long entry among single tokens, and lengths of every size
                        for (int i = 0; i < 300; ++i) nq[i] = i % 7 == 3 ? t * (i % 49 == 3 ? 40 : 1) : 1;
                        CHECK(gh_kv8_attention(kv, 300, seqs.data(), nq.data(), P, group * nkv, window, P) == GH_OK);
                        CHECK(all(nq, 300));
                    }
            std::vector<int32_t> none(300, 0);
            launches = 0;
            CHECK(gh_kv8_truncate(kv, 300, seqs.data(), none.data()) == GH_OK);
            // tokens of one long and many short sequences: not a grid of the long one's size for each
            for (int i = 0; i < 300; ++i) lens[i] = i == 5 ? max_seq : 1;
            CHECK(gh_kv8_append(kv, 300, seqs.data(), lens.data(), P, P) == GH_OK && all(lens, 300));
            CHECK(launches == (max_seq >= 5000 || (max_seq == 700 && nkv > 1) ? 3 : 2));
            launches = 1001;
            CHECK(gh_kv8_destroy(kv) == GH_OK);
        }
    }
    CHECK(gh_ctx_destroy(ctx) == GH_OK);
    CHECK(bad_launches == 0 && launches > 1000 && hip_stub_live_bytes() == 0);
    return 0;
}

// A cache outlives its context's destroy, and the last handle frees it.
int lifetimes() {
    gh_ctx* ctx = nullptr;
    const int32_t s[] = {0}, one[] = {1};
    for (int order = 0; order < 2; ++order) {
        gh_kv8 *a = nullptr, *b = nullptr;
        CHECK(gh_ctx_create(0, &ctx) == GH_OK && cache(ctx, 1, 64, 1, 64, &a) == GH_OK && cache(ctx, 1, 64, 1, 64, &b) == GH_OK);
        if (order == 0) CHECK(gh_ctx_destroy(ctx) == GH_OK);
        CHECK(gh_kv8_append(a, 1, s, one, P, P) == GH_OK && length(a, 0) == 1);
        CHECK(gh_kv8_destroy(a) == GH_OK);
        CHECK(gh_kv8_append(b, 1, s, one, P, P) == GH_OK);
        gh_kv8_release(b);
        if (order == 1) CHECK(gh_ctx_destroy(ctx) == GH_OK);
        CHECK(hip_stub_live_bytes() == 0);
    }
    // calls of two threads on one context, one of them creating and destroying
    CHECK(gh_ctx_create(0, &ctx) == GH_OK);
    gh_kv8* kv = nullptr;
    CHECK(cache(ctx, 1, 4096, 1, 64, &kv) == GH_OK);
    int other = 0;
    std::thread th([&] {
        for (int i = 0; i < 500; ++i) {
            gh_kv8* x = nullptr;
            if (gh_kv8_create(ctx, 1, 4096, 1, 64, &x) != GH_OK || gh_kv8_append(x, 1, s, one, P, P) != GH_OK ||
                gh_kv8_destroy(x) != GH_OK)
                other = 1;
        }
    });
    int mine = 0;
    for (int i = 0; i < 1000; ++i)
        if (gh_kv8_append(kv, 1, s, one, P, P) != GH_OK) mine = 1;
    th.join();
    CHECK(mine == 0 && other == 0 && length(kv, 0) == 1000);
    CHECK(gh_kv8_destroy(kv) == GH_OK && gh_ctx_destroy(ctx) == GH_OK && hip_stub_live_bytes() == 0);
    return 0;
}

}  // namespace

int main(int argc, char** argv) {
    static_assert(sizeof(gh_sampling) == 20, "five 4-byte fields, as the Python record");
    const char* mode = argc > 1 ? argv[1] : "";
    if (!std::strcmp(mode, "refusals")) return refusals();
    if (!std::strcmp(mode, "splits")) return splits();
    if (!std::strcmp(mode, "lifetimes")) return lifetimes();
    return 2;
}
