// Host side of the 8-bit KV cache: the handle, the checks of its calls and
// the split of an attention call into workgroups.
#include <algorithm>
#include <memory>
#include <new>

#include "host.h"
#include "kv8.h"

using namespace gh;

namespace {

constexpr int MAX_SEQ = 1 << 22;   // tokens a sequence
constexpr int MAX_ROWS = 1 << 20;  // query rows a kv head and sequence
constexpr int MAX_GROUP = 1024;    // heads a kv head: rows * group stays below 2^32 (Att8::group_inv)
constexpr int WASTE = 4096;        // empty workgroups that cost about what another launch does
constexpr int64_t MAX_QUERIES = 1 << 27;  // query rows of a sequence, all heads: 2^23 tiles
constexpr int64_t MAX_GRID = (1 << 24) - 1;  // workgroups of 256 threads in a grid's x (below 2^32 threads)

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

Kv8Dev dev(const gh_kv8* kv) { return {kv->kc, kv->vc, kv->ks, kv->vs, kv->kt, kv->vt, kv->nkv, kv->nb}; }

// The host arrays of a call: present, and every sequence known.
int check_seqs(const char* fn, const gh_kv8* kv, int32_t n, const int32_t* seqs, const int32_t* a, const int32_t* b) {
    if (n < 0 || (n > 0 && (!seqs || !a || !b))) return set_error(GH_ERR_INVALID, "%s: bad arguments", fn);
    for (int i = 0; i < n; ++i)
        if (seqs[i] < 0 || seqs[i] >= kv->n_seq)
            return set_error(GH_ERR_INVALID, "%s: sequence %d outside [0, %d)", fn, seqs[i], kv->n_seq);
    return GH_OK;
}

// No sequence twice (calls that change them).
int check_once(const char* fn, gh_kv8* kv, int32_t n, const int32_t* seqs) {
    if (++kv->call == INT32_MAX) {
        std::fill(kv->mark.begin(), kv->mark.end(), 0);
        kv->call = 1;
    }
    for (int i = 0; i < n; ++i) {
        if (kv->mark[seqs[i]] == kv->call) return set_error(GH_ERR_INVALID, "%s: sequence %d twice", fn, seqs[i]);
        kv->mark[seqs[i]] = kv->call;
    }
    return GH_OK;
}

// Calls that change the cache's length, which the host keeps, cannot be
// replayed from a graph.
int check_not_capturing(const char* fn, gh_ctx* ctx) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    GH_HIP(hipStreamIsCapturing(ctx->stream, &st));
    if (st != hipStreamCaptureStatusNone)
        return set_error(GH_ERR_STATE, "%s changes the cache's length and cannot be captured", fn);
    return GH_OK;
}

// Blocks a workgroup of the attention takes at most.  `most`: of the longest
// tile; `work`: of all `wgs` (entry, kv head, row tile) together.  A kv head's
// keys are cut into chunks where there are too few workgroups to fill the
// device, which costs a second launch of 4 us to join them.  Call times in us,
// 128 dims and 8 kv heads unless said otherwise:
//  - tile 4, a wave a block, eight of them side by side: uncut up to 16 blocks
//    (1024 tokens, 256 dims: 21, by eights 23), or where the uncut workgroups
//    fill the device in nearly whole rounds (32 sequences of 4096: 56, cut in
//    two 60), if the longest is not far from the average; else as many chunks
//    as fill it once, of 8 blocks at least (one sequence of 131072 tokens: 58,
//    by eights 73, uncut 589; 64 of 4096 with one head of 256 dims: 39, by
//    eights 43, uncut 57), or of 4 while these leave CUs to fill: a CU's share
//    of the bandwidth counts (32768 tokens of one head of 256 dims: 23, by
//    eights 25; 131072 of it 35 and 29).
//  - tile 16, four blocks a step: uncut up to two steps (a prompt of 300: 23,
//    by fours 27) or from a workgroup a CU on (64 sequences of 1024, 4 tokens
//    each: 29, in halves 36; a prompt of 1024: 30, in halves 47), but for long
//    ones short of two a CU (16 sequences of 32768 with drafts of 5: 225 by 64
//    blocks, 285 uncut); else as many as fill it twice (one of 32768 with a
//    draft of 5: 34, by fours 43, uncut 240).
int kv8_chunk(int hd, int tile, int most, int64_t work, int64_t wgs) {
    const bool even = most * wgs <= 2 * work;
    auto fill = [&](int64_t n, int least) { return (int)std::max<int64_t>(least, (work + n - 1) / n); };
    if (tile == 4) {
        const int64_t slots = hd <= 64 ? 512 : 256, rounds = (wgs + slots - 1) / slots;
        return most <= 16 || (wgs * 10 >= 9 * rounds * slots && even) ? std::max(most, 1) : fill(slots, work <= 1024 ? 4 : 8);
    }
    if (most <= 8 || (even && wgs >= (most <= 64 ? 256 : 512))) return std::max(most, 1);
    return wgs < 256 ? fill(512, 4) : fill(2048, 64);
}

int blocks_of(int begin, int end) {  // blocks that [begin, end) touches
    return end > begin ? (end - 1) / KV8_BLOCK - begin / KV8_BLOCK + 1 : 0;
}

// One entry of an append, a read or an attention.
struct Entry {
    int seq, pos, off, cnt;  // as in Kv8Batch
    int x, y;                // extents in the grid
    int blocks;              // attention: of keys
};

void to_batch(const Entry* e, int n, Kv8Batch& b) {
    int part = 0;
    for (int i = 0; i < n; ++i) {
        b.seq[i] = e[i].seq;
        b.pos[i] = e[i].pos;
        b.off[i] = e[i].off;
        b.cnt[i] = e[i].cnt;
        b.part[i] = part;
        part += e[i].cnt;
    }
}

// launch(entries, n) of the entries that have tokens, in launches of like
// sizes: a grid has as many workgroups for each as for the largest, so that
// small ones beside a large one would be passed over in empty workgroups, a
// microsecond a thousand.  A prompt of 16384 tokens among 239 single ones is
// appended in 591 us by one launch, in 107 so.  A size is the product of two
// extents of the grid; `heads` is its third.
template <class F>
int launch_by_size(Entry* e, int n, int64_t heads, F&& launch) {
    n = (int)(std::remove_if(e, e + n, [](const Entry& x) { return x.cnt == 0; }) - e);
    auto wasted = [&](int64_t grid, int64_t sum) { return (grid - sum) * heads > std::max<int64_t>(sum * heads, WASTE); };
    int64_t x = 0, y = 0, sum = 0;
    for (int i = 0; i < n; ++i) {
        x = std::max<int64_t>(x, e[i].x);
        y = std::max<int64_t>(y, e[i].y);
        sum += (int64_t)e[i].x * e[i].y;
    }
    if (n == 0 || !wasted(x * y * n, sum)) return n ? launch(e, n) : GH_OK;
    std::stable_sort(e, e + n, [](const Entry& a, const Entry& b) { return (int64_t)a.x * a.y > (int64_t)b.x * b.y; });
    for (int at = 0, end; at < n; at = end) {
        x = y = sum = 0;
        for (end = at; end < n; ++end) {
            const int64_t x1 = std::max<int64_t>(x, e[end].x), y1 = std::max<int64_t>(y, e[end].y);
            const int64_t sum1 = sum + (int64_t)e[end].x * e[end].y;
            if (end > at && wasted(x1 * y1 * (end + 1 - at), sum1)) break;
            x = x1;
            y = y1;
            sum = sum1;
        }
        GH_CHECK(launch(e + at, end - at));
    }
    return GH_OK;
}

int most_blocks(const Entry* e, int n) {
    int most = 0;
    for (int i = 0; i < n; ++i) most = std::max(most, e[i].x);
    return most;
}

// Key blocks that a row tile of the entry may see: up to the window and the
// tile's own rows.
int keys_of(const Entry& e, const Att8& a, int tile) {
    const int span = a.window ? (int)std::min<int64_t>(e.pos, (int64_t)a.window + tile / a.group + 1) : e.pos;
    return std::min((e.pos + KV8_BLOCK - 1) / KV8_BLOCK, span / KV8_BLOCK + 2);
}

int tiles_of(const Entry& e, const Att8& a, int tile) { return (e.cnt * a.group + tile - 1) / tile; }

// Sums over some entries, whose blocks and row tiles are set, and the chunks
// that follow.
struct Work {
    int most = 0, tiles = 0;    // blocks of the longest row tile, tiles of the longest entry
    int64_t work = 0, wgs = 0;  // blocks of all row tiles, and these
    int chunk = 1;
    Work(const gh_kv8* kv, const Entry* e, int n, int tile) {
        for (int i = 0; i < n; ++i) {
            most = std::max(most, e[i].blocks);
            tiles = std::max(tiles, e[i].x);
            wgs += (int64_t)e[i].x * kv->nkv;
            work += (int64_t)e[i].x * kv->nkv * e[i].blocks;
        }
        chunk = kv8_chunk(kv->hd, tile, most, work, wgs);
    }
    int parts(int blocks) const { return std::max(1, (blocks + chunk - 1) / chunk); }
};

// One launch (and one that joins the chunks) for entries with query tokens.
int attention_launch(gh_kv8* kv, Entry* e, int n, int tile, Att8 a) {
    Work w(kv, e, n, tile);
    for (int i = 0; i < n; ++i) {
        a.most_q = std::max(a.most_q, e[i].cnt);
        a.rows += (size_t)e[i].cnt * a.heads;
    }
    // nothing to join where a grid would be too large for it
    if ((int64_t)a.most_q * a.heads * (kv->hd / 32) > MAX_GRID || (int64_t)w.parts(w.most) * w.tiles * kv->nkv > MAX_GRID)
        w.chunk = std::max(w.most, 1);
    a.tile = tile;
    a.tiles = w.tiles;
    a.chunk = w.chunk;
    a.ns = w.parts(w.most);
    if (a.ns > 1) {
        void* part = nullptr;
        GH_CHECK(ctx_scratch(kv->ctx, a.rows * a.ns * (kv->hd + 2) * sizeof(float), &part));
        a.part = (float*)part;
    }
    // the longest first: their workgroups start before the others'
    std::stable_sort(e, e + n, [](const Entry& x, const Entry& y) { return x.blocks > y.blocks; });
    Kv8Batch b;
    to_batch(e, n, b);
    return launch_kv8_attention(dev(kv), kv->hd, b, n, a, kv->ctx->stream);
}

int attention_launches(gh_kv8* kv, Entry* e, int n, int tile, const Att8& a) {
    for (int i = 0; i < n; ++i) {
        e[i].x = tiles_of(e[i], a, tile);
        e[i].blocks = keys_of(e[i], a, tile);
    }
    const Work w(kv, e, n, tile);
    for (int i = 0; i < n; ++i) e[i].y = w.parts(e[i].blocks);
    return launch_by_size(e, n, kv->nkv, [&](Entry* x, int c) { return attention_launch(kv, x, c, tile, a); });
}

// Entries of up to four query rows a kv head (decoding) have a kernel of their
// own, but join the others where one row tile holds any of these (drafts): 64
// sequences of 4096 tokens, half of them with drafts of 4, take 97 us joined
// and 111 apart.  Beside a prompt they would be passed over by most of the
// grid: 63 of them and a prompt of 16 tokens 196 us joined, 102 apart.
int attention_batch(gh_kv8* kv, Entry* e, int n, const Att8& a) {
    n = (int)(std::remove_if(e, e + n, [](const Entry& x) { return x.cnt == 0; }) - e);
    Entry* wide = std::stable_partition(e, e + n, [&](const Entry& x) { return x.cnt * a.group <= 4; });
    if (std::all_of(wide, e + n, [&](const Entry& x) { return tiles_of(x, a, 16) == 1; }) && wide < e + n) wide = e;
    GH_CHECK(attention_launches(kv, e, (int)(wide - e), 4, a));
    return attention_launches(kv, wide, (int)(e + n - wide), 16, a);
}

}  // namespace

gh_kv8::~gh_kv8() {
    if (mem) hipFree(mem);
}

extern "C" int gh_kv8_create(gh_ctx* ctx, int32_t n_seq, int32_t max_seq, int32_t n_kv_heads, int32_t head_dim,
                             gh_kv8** out) {
    GH_CHECK(ctx_bind(ctx));
    if (!out) return set_error(GH_ERR_INVALID, "gh_kv8_create: null output");
    if (n_seq <= 0 || n_seq > (1 << 20) || max_seq <= 0 || max_seq > MAX_SEQ || n_kv_heads <= 0 || n_kv_heads > 1024)
        return set_error(GH_ERR_INVALID, "gh_kv8_create: bad shape (%d sequences of %d tokens, %d kv heads)", n_seq,
                         max_seq, n_kv_heads);
    if (head_dim != 32 && head_dim != 64 && head_dim != 128 && head_dim != 256)
        return set_error(GH_ERR_INVALID, "gh_kv8_create: head_dim %d is not 32, 64, 128 or 256", head_dim);
    Lock lk(ctx->mu);
    std::unique_ptr<gh_kv8> kv(new (std::nothrow) gh_kv8);
    if (!kv) return set_error(GH_ERR_OOM, "gh_kv8_create: host memory");
    kv->ctx = ctx;
    kv->n_seq = n_seq;
    kv->max_seq = max_seq;
    kv->nkv = n_kv_heads;
    kv->hd = head_dim;
    kv->nb = (max_seq + KV8_BLOCK - 1) / KV8_BLOCK;
    const size_t heads = (size_t)n_seq * n_kv_heads, blocks = heads * kv->nb;
    struct {
        void** p;
        size_t bytes;
    } parts[] = {{(void**)&kv->kc, blocks * KV8_BLOCK * kv8_k_row(head_dim)},
                 {(void**)&kv->vc, blocks * KV8_BLOCK * head_dim},
                 {(void**)&kv->ks, blocks * 4},
                 {(void**)&kv->vs, blocks * 4},
                 {(void**)&kv->kt, heads * KV8_BLOCK * head_dim * 4},
                 {(void**)&kv->vt, heads * KV8_BLOCK * head_dim * 4}};
    size_t total = 0;
    for (auto& p : parts) total += (p.bytes + 255) / 256 * 256;
    hipError_t e = hipMalloc(&kv->mem, total);
    if (e != hipSuccess) {
        kv->mem = nullptr;
        return set_error(GH_ERR_OOM, "gh_kv8_create: hipMalloc(%zu): %s", total, hipGetErrorString(e));
    }
    char* at = (char*)kv->mem;
    for (auto& p : parts) {
        *p.p = at;
        at += (p.bytes + 255) / 256 * 256;
    }
    try {
        kv->len.assign(n_seq, 0);
        kv->mark.assign(n_seq, 0);
        ctx->kv8s.push_back(kv.get());
    } catch (const std::bad_alloc&) {  // no exception leaves a C entry
        return set_error(GH_ERR_OOM, "gh_kv8_create: host memory for %d sequences", n_seq);
    }
    *out = kv.release();
    handle_add(*out, HK_KV8);
    return GH_OK;
}

extern "C" int gh_kv8_destroy(gh_kv8* kv) {
    if (!kv) return GH_OK;
    if (!handle_take(kv, HK_KV8)) return dead_handle("gh_kv8_destroy", HK_KV8);
    gh_ctx* ctx = kv->ctx;
    bool dead = false;
    {
        Lock lk(ctx->mu);
        hipSetDevice(ctx->device);
        hipStreamSynchronize(ctx->stream);
        auto& v = ctx->kv8s;
        v.erase(std::remove(v.begin(), v.end(), kv), v.end());
        delete kv;
        dead = ctx_dead(ctx);
    }
    if (dead) ctx_free(ctx);
    return GH_OK;
}

extern "C" void gh_kv8_release(gh_kv8* kv) { gh_kv8_destroy(kv); }

extern "C" int gh_kv8_length(gh_kv8* kv, int32_t seq, int32_t* len_out) {
    GH_LIVE(kv, HK_KV8);
    if (!len_out) return set_error(GH_ERR_INVALID, "gh_kv8_length: null output");
    Lock lk(kv->ctx->mu);
    if (seq < 0 || seq >= kv->n_seq)
        return set_error(GH_ERR_INVALID, "gh_kv8_length: sequence %d outside [0, %d)", seq, kv->n_seq);
    *len_out = kv->len[seq];
    return GH_OK;
}

extern "C" int gh_kv8_append(gh_kv8* kv, int32_t n, const int32_t* seqs, const int32_t* n_tok, const float* k,
                             const float* v) {
    GH_LIVE(kv, HK_KV8);
    gh_ctx* ctx = kv->ctx;
    GH_CHECK(dev_bind(ctx));
    Lock lk(ctx->mu);
    GH_CHECK(check_seqs("gh_kv8_append", kv, n, seqs, n_tok, n_tok));
    GH_CHECK(check_once("gh_kv8_append", kv, n, seqs));
    int64_t total = 0;
    for (int i = 0; i < n; ++i) {
        if (n_tok[i] < 0) return set_error(GH_ERR_INVALID, "gh_kv8_append: %d tokens", n_tok[i]);
        if (n_tok[i] > kv->max_seq - kv->len[seqs[i]])
            return set_error(GH_ERR_RANGE, "gh_kv8_append: %d tokens behind %d of sequence %d pass max_seq %d", n_tok[i],
                             kv->len[seqs[i]], seqs[i], kv->max_seq);
        total += n_tok[i];
    }
    if (total == 0) return GH_OK;
    if (!k || !v || !aligned(k) || !aligned(v))
        return set_error(GH_ERR_INVALID, "gh_kv8_append: k and v must be 16-byte aligned device pointers");
    GH_CHECK(check_not_capturing("gh_kv8_append", ctx));
    const size_t row = (size_t)kv->nkv * kv->hd;
    for (int i0 = 0; i0 < n; i0 += KV8_BATCH) {
        const int m = std::min(n - i0, KV8_BATCH);
        Entry e[KV8_BATCH];
        int rows = 0;
        for (int i = 0; i < m; ++i) {
            const int s = seqs[i0 + i], t = n_tok[i0 + i];
            e[i] = {s, kv->len[s], rows, t, blocks_of(kv->len[s], kv->len[s] + t), 1, 0};
            rows += t;
        }
        GH_CHECK(launch_by_size(e, m, 2 * kv->nkv, [&](const Entry* x, int c) {
            Kv8Batch b;
            to_batch(x, c, b);
            return launch_kv8_append(dev(kv), kv->hd, b, c, most_blocks(x, c), k, v, ctx->stream);
        }));
        k += (size_t)rows * row;
        v += (size_t)rows * row;
    }
    for (int i = 0; i < n; ++i) kv->len[seqs[i]] += n_tok[i];
    return op_sync(ctx);
}

extern "C" int gh_kv8_truncate(gh_kv8* kv, int32_t n, const int32_t* seqs, const int32_t* lens) {
    GH_LIVE(kv, HK_KV8);
    gh_ctx* ctx = kv->ctx;
    GH_CHECK(dev_bind(ctx));
    Lock lk(ctx->mu);
    GH_CHECK(check_seqs("gh_kv8_truncate", kv, n, seqs, lens, lens));
    GH_CHECK(check_once("gh_kv8_truncate", kv, n, seqs));
    for (int i = 0; i < n; ++i)
        if (lens[i] < 0 || lens[i] > kv->len[seqs[i]])
            return set_error(GH_ERR_RANGE, "gh_kv8_truncate: sequence %d holds %d tokens, not %d", seqs[i],
                             kv->len[seqs[i]], lens[i]);
    GH_CHECK(check_not_capturing("gh_kv8_truncate", ctx));
    bool ran = false;
    for (int i0 = 0; i0 < n; i0 += KV8_BATCH) {
        // only sequences that end inside a block afterwards have anything to redo
        Kv8Batch b;
        int m = 0;
        for (int i = i0; i < std::min(n, i0 + KV8_BATCH); ++i) {
            if (lens[i] == kv->len[seqs[i]] || lens[i] % KV8_BLOCK == 0) continue;
            b.seq[m] = seqs[i];
            b.pos[m] = kv->len[seqs[i]];
            b.off[m] = 0;
            b.cnt[m++] = lens[i];
        }
        if (m) GH_CHECK(launch_kv8_truncate(dev(kv), kv->hd, b, m, ctx->stream));
        ran = ran || m;
    }
    for (int i = 0; i < n; ++i) kv->len[seqs[i]] = lens[i];
    return ran ? op_sync(ctx) : GH_OK;
}

extern "C" int gh_kv8_read(gh_kv8* kv, int32_t n, const int32_t* seqs, const int32_t* begins, const int32_t* ends,
                           float* k_out, float* v_out) {
    GH_LIVE(kv, HK_KV8);
    gh_ctx* ctx = kv->ctx;
    GH_CHECK(dev_bind(ctx));
    Lock lk(ctx->mu);
    GH_CHECK(check_seqs("gh_kv8_read", kv, n, seqs, begins, ends));
    int64_t total = 0;
    for (int i = 0; i < n; ++i) {
        if (begins[i] < 0 || ends[i] < begins[i] || ends[i] > kv->len[seqs[i]])
            return set_error(GH_ERR_RANGE, "gh_kv8_read: tokens [%d, %d) of sequence %d, which holds %d", begins[i],
                             ends[i], seqs[i], kv->len[seqs[i]]);
        total += ends[i] - begins[i];
    }
    if (total == 0 || (!k_out && !v_out)) return GH_OK;
    if (!aligned(k_out) || !aligned(v_out))
        return set_error(GH_ERR_INVALID, "gh_kv8_read: k_out and v_out must be 16-byte aligned device pointers");
    const size_t row = (size_t)kv->nkv * kv->hd;
    for (int i0 = 0; i0 < n; i0 += KV8_BATCH) {
        const int m = std::min(n - i0, KV8_BATCH);
        Entry e[KV8_BATCH];
        int rows = 0;
        for (int i = 0; i < m; ++i) {
            const int at = begins[i0 + i], end = ends[i0 + i];
            e[i] = {seqs[i0 + i], at, rows, end - at, blocks_of(at, end), 1, 0};
            rows += end - at;
        }
        GH_CHECK(launch_by_size(e, m, 2 * kv->nkv, [&](const Entry* x, int c) {
            Kv8Batch b;
            to_batch(x, c, b);
            return launch_kv8_read(dev(kv), kv->hd, b, c, most_blocks(x, c), k_out, v_out, ctx->stream);
        }));
        if (k_out) k_out += (size_t)rows * row;
        if (v_out) v_out += (size_t)rows * row;
    }
    return op_sync(ctx);
}

extern "C" int gh_kv8_attention(gh_kv8* kv, int32_t n, const int32_t* seqs, const int32_t* n_q, const float* q,
                                int32_t n_heads, int32_t window, float* out) {
    GH_LIVE(kv, HK_KV8);
    gh_ctx* ctx = kv->ctx;
    GH_CHECK(dev_bind(ctx));
    Lock lk(ctx->mu);
    GH_CHECK(check_seqs("gh_kv8_attention", kv, n, seqs, n_q, n_q));
    if (n_heads <= 0 || n_heads % kv->nkv || window < 0)
        return set_error(GH_ERR_INVALID, "gh_kv8_attention: %d heads over %d kv heads, window %d", n_heads, kv->nkv, window);
    const int group = n_heads / kv->nkv;
    if (group > MAX_GROUP) return set_error(GH_ERR_RANGE, "gh_kv8_attention: %d heads a kv head", group);
    int64_t total = 0;
    for (int i = 0; i < n; ++i) {
        if (n_q[i] < 0) return set_error(GH_ERR_INVALID, "gh_kv8_attention: %d query tokens", n_q[i]);
        if ((int64_t)n_q[i] * group > MAX_ROWS || (int64_t)n_q[i] * n_heads > MAX_QUERIES)
            return set_error(GH_ERR_RANGE, "gh_kv8_attention: %d query tokens of %d heads a kv head", n_q[i], group);
        total += n_q[i];
    }
    if (total == 0) return GH_OK;
    if (!q || !out || !aligned(q) || !aligned(out))
        return set_error(GH_ERR_INVALID, "gh_kv8_attention: q and out must be 16-byte aligned device pointers");
    Att8 a{};
    a.heads = n_heads;
    a.group = group;
    a.group_inv = group == 1 ? 0 : (unsigned)(((uint64_t(1) << 32) + group - 1) / group);
    a.window = window >= kv->max_seq ? 0 : window;
    a.q = q;
    a.out = out;
    for (int i0 = 0; i0 < n; i0 += KV8_BATCH) {
        const int m = std::min(n - i0, KV8_BATCH);
        Entry e[KV8_BATCH];
        int tokens = 0;
        for (int i = 0; i < m; ++i) {
            const int s = seqs[i0 + i], t = n_q[i0 + i];
            e[i] = {s, kv->len[s], tokens, t, 0, 0, 0};
            tokens += t;
        }
        GH_CHECK(attention_batch(kv, e, m, a));
        a.q += (size_t)tokens * n_heads * kv->hd;
        a.out += (size_t)tokens * n_heads * kv->hd;
    }
    return op_sync(ctx);
}
