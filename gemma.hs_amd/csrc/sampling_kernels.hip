// gfx950 kernels of the batched sampler (temperature, top-k, top-p, min-p).
//
// The draw is a search along the ranks: for the top_k-th element, for the
// first whose running mass reaches top_p of what top_k left, for the first
// below min_p, and for the first whose running mass passes u times what the
// three leave.  None needs the row sorted:
//   1. largest and smallest logit (k_smp_stat),
//   2. a histogram over SMP_BINS equal steps of the logit between them, with
//      the number and the mass of each bin's elements (k_smp_hist): sums over
//      its bins say in which bin, or few bins, each search ends,
//   3. the elements of those bins, a list (k_smp_gather),
//   4. the list sorted, its running mass on top of the bins' in front of it:
//      the exact answers (k_smp_pick).
// A list that does not fit (rows with thousands of equal logits) is searched
// digit by digit instead (slow_row).  Rows that one workgroup reads quickly
// run all four steps in one kernel (k_smp_row).
#include <hip/hip_runtime.h>

#include "sampling.h"

namespace gh {

namespace {

constexpr int NT = 1024;
constexpr int NW = NT / 64;

typedef unsigned long long u64;

// Ascending in rank order: value descending, then index ascending.
__device__ __forceinline__ uint32_t value_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);  // -0 ranks as 0
    return (b & 0x80000000u) ? b : ~(b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k : ~k & 0x7fffffffu);
}
__device__ __forceinline__ u64 rank_key(float v, int i) { return ((u64)value_key(v) << 32) | (unsigned)i; }

// A row's weights exp((l - max) / T), as integers of smp_bits fractional bits:
// their sums do not depend on the order, and are exact to 2^-bits a weight.
// In 64 bits because a draw compares sums over the whole vocabulary.
struct Weights {
    float top;
    double inv_t, one;
    __device__ __forceinline__ double real(float l) const {
        return l == top ? 1.0 : exp(((double)l - (double)top) * inv_t);
    }
    __device__ __forceinline__ u64 fixed(float l) const { return (u64)__double2ull_rn(real(l) * one); }
};

// What the bins are: equal steps of top - l up to `reach`, behind which every
// weight is zero.  Monotonic in l, so that bins follow the ranks.
struct Bins {
    float top, scale, reach;
    __device__ __forceinline__ bool in_reach(float l) const { return l == top || top - l <= reach; }
    __device__ __forceinline__ int of(float l) const {
        return l == top ? 0 : (int)fminf((top - l) * scale, (float)(SMP_BINS - 1));
    }
};

__device__ __forceinline__ u64 shfl_xor64(u64 v, int o) {
    const unsigned lo = __shfl_xor((unsigned)v, o, 64), hi = __shfl_xor((unsigned)(v >> 32), o, 64);
    return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ u64 shfl_up64(u64 v, int o) {
    const unsigned lo = __shfl_up((unsigned)v, o, 64), hi = __shfl_up((unsigned)(v >> 32), o, 64);
    return ((u64)hi << 32) | lo;
}

struct Range {
    int lo, hi;
    __device__ __forceinline__ bool has(int b) const { return b >= lo && b <= hi; }
};

struct Shared {
    u64 mass[SMP_BINS];       // per bin, then running
    unsigned count[SMP_BINS];
    u64 list[SMP_LIST];
    u64 red[NW];
    unsigned red32[NW];
    u64 key, base_mass;  // slow_row
    unsigned base_count;
    unsigned n_list;
    int at;
    u64 found;
    int bin[8];
    u64 before[8], upto[8];
};

template <class Op>
__device__ u64 block_reduce(u64 v, Shared& sh, Op op) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = op(v, shfl_xor64(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh.red[threadIdx.x & (NW - 1)];
#pragma unroll
    for (int o = NW / 2; o > 0; o >>= 1) v = op(v, shfl_xor64(v, o));
    return v;
}

// inclusive running sums over the threads; *total the last
__device__ __forceinline__ void block_scan(u64& m, unsigned& c, Shared& sh) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 a = shfl_up64(m, o);
        const unsigned b = __shfl_up(c, o, 64);
        if (lane >= o) m += a, c += b;
    }
    __syncthreads();
    if (lane == 63) sh.red[w] = m, sh.red32[w] = c;
    __syncthreads();
    u64 pm = 0;
    unsigned pc = 0;
    for (int i = 0; i < w; ++i) pm += sh.red[i], pc += sh.red32[i];
    m += pm;
    c += pc;
}

// ------------------------------------------------------------------
// step 1
// ------------------------------------------------------------------
struct Stat {
    u64 first;  // rank key of the first in rank order; ~0: nothing above -inf
    float low;  // smallest value above -inf
    bool nan;
};

// f(index, logit) of the elements [i0, i1), several loads in flight a thread
template <class F>
__device__ __forceinline__ void each_logit(const float* l, int i0, int i1, F&& f) {
    constexpr int U = 8;
    int i = i0 + threadIdx.x;
    for (; i + (U - 1) * NT < i1; i += U * NT) {
        float v[U];
#pragma unroll
        for (int j = 0; j < U; ++j) v[j] = l[i + j * NT];
#pragma unroll
        for (int j = 0; j < U; ++j) f(i + j * NT, v[j]);
    }
    for (; i < i1; i += NT) f(i, l[i]);
}

__device__ __forceinline__ Stat range_stat(const float* l, int i0, int i1, Shared& sh) {
    u64 first = ~0ull;
    float low = INFINITY;
    unsigned nan = 0;
    each_logit(l, i0, i1, [&](int i, float v) {
        nan |= v != v;
        if (v > -INFINITY) {
            first = min(first, rank_key(v, i));
            low = fminf(low, v);
        }
    });
    first = block_reduce(first, sh, [](u64 a, u64 b) { return a < b ? a : b; });
    // smallest value = largest value key; the NaN flag in the bit above it
    const u64 rest = block_reduce(((u64)nan << 32) | (low < INFINITY ? value_key(low) : 0u), sh, [](u64 a, u64 b) {
        return ((a | b) & (1ull << 32)) | max((unsigned)a, (unsigned)b);
    });
    return {first, key_value((unsigned)rest), (rest >> 32) != 0};
}

// One step behind the stats: true if the row's token is known (written).
__device__ __forceinline__ bool settled(const Stat& s, const gh_sampling& rule, int32_t* token) {
    const bool bad = s.nan || s.first == ~0ull;
    if (!bad && rule.temperature > 0.0f) return false;
    if (threadIdx.x == 0) *token = bad ? -1 : (int)(unsigned)s.first;
    return true;
}

__device__ __forceinline__ Weights weights_of(const Stat& s, const gh_sampling& rule, double one) {
    return {key_value((unsigned)(s.first >> 32)), 1.0 / (double)rule.temperature, one};
}

// `dead`: (top - l) / T from which on a weight rounds to zero
__device__ __forceinline__ Bins bins_of(const Stat& s, const Weights& w, double dead) {
    const double d = min((double)w.top - (double)s.low, dead / w.inv_t);
    if (!(d > 0.0)) return {w.top, 0.0f, 0.0f};  // one value (an infinite one among them): one bin
    return {w.top, (float)fmin((double)SMP_BINS / d, 3e38), (float)fmin(d * 1.000001, 3.4e38)};
}

// ------------------------------------------------------------------
// step 2
// ------------------------------------------------------------------
__device__ __forceinline__ void clear_bins(Shared& sh) {
    for (int b = threadIdx.x; b < SMP_BINS; b += NT) sh.mass[b] = 0, sh.count[b] = 0;
    if (threadIdx.x == 0) sh.n_list = 0;
    __syncthreads();
}

__device__ __forceinline__ void range_hist(const float* l, int i0, int i1, const Weights& w, const Bins& bins, bool counts,
                                           Shared& sh) {
    each_logit(l, i0, i1, [&](int, float v) {
        if (!bins.in_reach(v)) return;
        const u64 m = w.fixed(v);
        if (!m) return;
        const int b = bins.of(v);
        atomicAdd(&sh.mass[b], m);
        if (counts) atomicAdd(&sh.count[b], 1u);
    });
    __syncthreads();
}

// ------------------------------------------------------------------
// step 3: where the searches end, from the bins alone
// ------------------------------------------------------------------
struct Cuts {
    bool k, p, m;        // which of the rules cut anything off
    u64 total;           // mass of all
    u64 upto_m;          // min_p: mass of the bins that it cannot reach behind
    Range at[4];         // bins whose elements decide: top_k, top_p, min_p, the draw
    __device__ __forceinline__ bool has(int b) const { return at[0].has(b) || at[1].has(b) || at[2].has(b) || at[3].has(b); }
};

// The bin in which a running sum first satisfies `reached`; slot i of sh.
template <class P>
__device__ __forceinline__ void find_bin(int i, Shared& sh, P&& reached) {
    for (int b = threadIdx.x; b < SMP_BINS; b += NT) {
        const bool here = reached(sh.mass[b], sh.count[b]);
        const bool there = b > 0 && reached(sh.mass[b - 1], sh.count[b - 1]);
        if (here && !there) {
            sh.bin[i] = b;
            sh.before[i] = b > 0 ? sh.mass[b - 1] : 0;
            sh.upto[i] = sh.mass[b];
        }
    }
}

// sh.mass, sh.count: per bin; running afterwards.
__device__ __forceinline__ Cuts find_cuts(const Weights& w, const Bins& bins, const gh_sampling& rule, Shared& sh) {
    static_assert(SMP_BINS == 2 * NT, "two bins a thread");
    const int tid = threadIdx.x;
    {
        const u64 m0 = sh.mass[2 * tid], m1 = sh.mass[2 * tid + 1];
        const unsigned c0 = sh.count[2 * tid], c1 = sh.count[2 * tid + 1];
        u64 m = m0 + m1;
        unsigned c = c0 + c1;
        block_scan(m, c, sh);
        sh.mass[2 * tid] = m - m1;
        sh.mass[2 * tid + 1] = m;
        sh.count[2 * tid] = c - c1;
        sh.count[2 * tid + 1] = c;
        __syncthreads();
    }
    Cuts q;
    q.total = sh.mass[SMP_BINS - 1];
    // what is behind the last element with a weight cannot be drawn: a top_k
    // that reaches there leaves all the mass
    const unsigned alive = sh.count[SMP_BINS - 1];
    q.k = rule.top_k > 0 && (unsigned)rule.top_k < alive;
    q.p = rule.top_p < 1.0f;
    q.m = rule.min_p > 0.0f;
    const Range none{1, 0};
    for (Range& r : q.at) r = none;
    u64 zlo = q.total, zhi = q.total;  // mass that top_k leaves
    if (q.k) {
        const unsigned k = rule.top_k;
        find_bin(0, sh, [&](u64, unsigned c) { return c >= k; });
        __syncthreads();
        q.at[0] = {sh.bin[0], sh.bin[0]};
        zlo = sh.before[0];
        zhi = sh.upto[0];
    }
    u64 lo = zlo, hi = zhi;  // mass that all three leave
    if (q.p) {
        const double tlo = (double)rule.top_p * (double)zlo, thi = (double)rule.top_p * (double)zhi;
        find_bin(1, sh, [&](u64 m, unsigned) { return m > 0 && (double)m >= tlo; });
        find_bin(2, sh, [&](u64 m, unsigned) { return m > 0 && (double)m >= thi; });
        __syncthreads();
        q.at[1] = {sh.bin[1], sh.bin[2]};
        lo = min(lo, sh.before[1]);
        hi = min(hi, sh.upto[2]);
    }
    q.upto_m = q.total;
    if (q.m) {
        // the logit at which a weight falls below min_p, a bin to either side for roundings
        const double d = -log((double)rule.min_p) / w.inv_t * (double)bins.scale;
        q.m = d < SMP_BINS + 1;  // else every weight reaches it
        if (q.m) {
            const int b = (int)d;
            q.at[2] = {max(b - 1, 0), min(b + 1, SMP_BINS - 1)};
            q.upto_m = sh.mass[q.at[2].hi];
            lo = min(lo, q.at[2].lo > 0 ? sh.mass[q.at[2].lo - 1] : 0);
            hi = min(hi, q.upto_m);
        }
    }
    const double ulo = (double)rule.u * (double)lo, uhi = (double)rule.u * (double)hi;
    find_bin(3, sh, [&](u64 m, unsigned) { return (double)m > ulo; });
    find_bin(4, sh, [&](u64 m, unsigned) { return (double)m > uhi; });
    __syncthreads();
    q.at[3] = {sh.bin[3], sh.bin[4]};
    return q;
}

__device__ __forceinline__ void range_gather(const float* l, int i0, int i1, const Bins& bins, const Cuts& cuts, u64* list,
                                             unsigned* n) {
    each_logit(l, i0, i1, [&](int i, float v) {
        if (!bins.in_reach(v) || !cuts.has(bins.of(v))) return;
        const unsigned at = atomicAdd(n, 1u);
        if (at < SMP_LIST) list[at] = rank_key(v, i);
    });
    __syncthreads();
}

// ------------------------------------------------------------------
// step 4
// ------------------------------------------------------------------
// ascending, in LDS; n <= SMP_LIST
__device__ __forceinline__ void sort_list(Shared& sh, int n) {
    int size = 64;
    while (size < n) size *= 2;
    for (int i = n + threadIdx.x; i < size; i += NT) sh.list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= size; k *= 2) {
        for (int j = k / 2; j > 0; j /= 2) {
            for (int t = threadIdx.x; t < size / 2; t += NT) {
                const int a = 2 * t - (t & (j - 1)), b = a + j;  // a has a 0 where b has a 1
                const u64 x = sh.list[a], y = sh.list[b];
                if ((x > y) == ((a & k) == 0)) sh.list[a] = y, sh.list[b] = x;
            }
            __syncthreads();
        }
    }
}

// The token, from the bins' running sums and the sorted list of the cuts' bins.
__device__ __forceinline__ int pick(const Weights& w, const Bins& bins, const gh_sampling& rule, const Cuts& cuts, int n,
                                    Shared& sh) {
    constexpr int PER = SMP_LIST / NT;
    const int tid = threadIdx.x;
    u64 upto[PER];       // running mass up to and with the element
    unsigned rank[PER];  // and its rank, from 1
    float val[PER];
    {
        u64 m[PER], s = 0;
        int b[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = tid * PER + j;
            val[j] = i < n ? key_value((unsigned)(sh.list[i] >> 32)) : 0.0f;
            m[j] = i < n ? w.fixed(val[j]) : 0;
            b[j] = i < n ? bins.of(val[j]) : 0;
            s += m[j];
        }
        u64 at = s;
        unsigned dummy = 0;
        block_scan(at, dummy, sh);
        at -= s;  // of the list in front of this thread
        // per bin: what its elements' running sums in the list lack
        u64 om[PER];
        unsigned oc[PER];
        bool head[PER];
        u64 run = at;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = tid * PER + j;
            head[j] = i < n && (i == 0 || bins.of(key_value((unsigned)(sh.list[i - 1] >> 32))) != b[j]);
            om[j] = head[j] ? (b[j] > 0 ? sh.mass[b[j] - 1] : 0) - run : 0;
            oc[j] = head[j] ? (b[j] > 0 ? sh.count[b[j] - 1] : 0) - i : 0;
            run += m[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (head[j]) sh.mass[b[j]] = om[j], sh.count[b[j]] = oc[j];
        __syncthreads();
        run = at;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = tid * PER + j;
            run += m[j];
            upto[j] = i < n ? sh.mass[b[j]] + run : 0;
            rank[j] = i < n ? sh.count[b[j]] + i + 1 : 0;
        }
    }
    // f(j) true: the first such element in rank order; sh.at its place, sh.found its running mass
    auto first = [&](auto&& f) {
        __syncthreads();
        if (tid == 0) sh.at = n;
        __syncthreads();
#pragma unroll
        for (int j = PER - 1; j >= 0; --j)
            if (tid * PER + j < n && f(j)) atomicMin(&sh.at, tid * PER + j);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (tid * PER + j == sh.at) sh.found = upto[j];
        __syncthreads();
    };
    u64 left = cuts.total;
    if (cuts.k) {
        first([&](int j) { return rank[j] == (unsigned)rule.top_k; });
        left = sh.found;
    }
    u64 kept = left;
    if (cuts.p) {
        const double t = (double)rule.top_p * (double)left;
        first([&](int j) { return (double)upto[j] >= t; });
        kept = min(kept, sh.found);
    }
    if (cuts.m) {
        kept = min(kept, cuts.upto_m);
        first([&](int j) { return w.real(val[j]) < (double)rule.min_p; });
        if (sh.at < n) kept = min(kept, sh.found - w.fixed(key_value((unsigned)(sh.list[sh.at] >> 32))));
    }
    const double t = (double)rule.u * (double)kept;
    first([&](int j) { return (double)upto[j] > t; });
    return (int)(unsigned)sh.list[sh.at];
}

// ------------------------------------------------------------------
// rows whose list is too long
// ------------------------------------------------------------------
// The first element in rank order whose running count reaches `k` (k > 0), or
// whose running mass reaches (strict: passes) `t`: digit by digit of its rank
// key, from the counts and masses of the 256 values of each digit among the
// elements that share the digits before.  The mass up to and with it goes to
// sh.base_mass, its key to sh.key.
__device__ void find(const float* l, int n, const Weights& w, unsigned k, double t, bool strict, Shared& sh) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid == 0) sh.key = sh.base_mass = 0, sh.base_count = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        if (shift == 24) continue;  // indexes are below 2^24
        if (tid < 256) sh.mass[tid] = 0, sh.count[tid] = 0;
        __syncthreads();
        const u64 prefix = sh.key;
        each_logit(l, 0, n, [&](int i, float v) {
            const u64 key = rank_key(v, i);
            if (shift < 56 && (key >> (shift + 8)) != (prefix >> (shift + 8))) return;
            const int d = (int)(key >> shift) & 255;
            atomicAdd(&sh.count[d], 1u);
            const u64 m = w.fixed(v);
            if (m) atomicAdd(&sh.mass[d], m);
        });
        __syncthreads();
        if (tid == 0) {
            u64 mass = sh.base_mass;
            unsigned count = sh.base_count;
            int d = 0;
            for (; d < 255; ++d) {
                const u64 m = mass + sh.mass[d];
                const unsigned c = count + sh.count[d];
                if (k ? c >= k : sh.count[d] && (strict ? (double)m > t : (double)m >= t)) break;
                mass = m;
                count = c;
            }
            sh.key = prefix | ((u64)d << shift);
            sh.base_mass = mass;
            sh.base_count = count;
        }
        __syncthreads();
    }
    if (tid == 0) sh.base_mass += w.fixed(l[(unsigned)sh.key]);
    __syncthreads();
}

__device__ __noinline__ int slow_row(const float* l, int n, const Weights& w, const gh_sampling& rule, Shared& sh) {
    u64 total = 0, at_least = 0;
    each_logit(l, 0, n, [&](int, float v) {
        const u64 m = w.fixed(v);
        total += m;
        if (w.real(v) >= (double)rule.min_p) at_least += m;
    });
    auto plus = [](u64 a, u64 b) { return a + b; };
    total = block_reduce(total, sh, plus);
    at_least = block_reduce(at_least, sh, plus);
    if (rule.top_k > 0 && rule.top_k < n) {
        find(l, n, w, rule.top_k, 0.0, false, sh);
        total = sh.base_mass;
    }
    u64 kept = min(total, at_least);
    if (rule.top_p < 1.0f) {
        find(l, n, w, 0, (double)rule.top_p * (double)total, false, sh);
        kept = min(kept, sh.base_mass);
    }
    find(l, n, w, 0, (double)rule.u * (double)kept, true, sh);
    return (int)(unsigned)sh.key;
}

// ------------------------------------------------------------------
// kernels
// ------------------------------------------------------------------
// one workgroup a row
__global__ __launch_bounds__(NT) void k_smp_row(const float* logits, int n, double one, double dead, SmpRules rules,
                                                int32_t* tokens) {
    __shared__ Shared sh;
    const gh_sampling rule = rules.r[blockIdx.x];
    const float* l = logits + (size_t)blockIdx.x * n;
    int32_t* token = tokens + blockIdx.x;
    const Stat s = range_stat(l, 0, n, sh);
    if (settled(s, rule, token)) return;
    const Weights w = weights_of(s, rule, one);
    const Bins bins = bins_of(s, w, dead);
    clear_bins(sh);
    range_hist(l, 0, n, w, bins, rule.top_k > 0, sh);
    const Cuts cuts = find_cuts(w, bins, rule, sh);
    range_gather(l, 0, n, bins, cuts, sh.list, &sh.n_list);
    int t;
    const unsigned listed = sh.n_list;
    if (listed <= SMP_LIST) {
        sort_list(sh, listed);
        t = pick(w, bins, rule, cuts, listed, sh);
    } else {
        t = slow_row(l, n, w, rule, sh);
    }
    if (threadIdx.x == 0) *token = t;
}

__device__ __forceinline__ int chunk_begin(int n, int c, int chunks) { return (int)((int64_t)n * c / chunks); }

// a row's chunks: stats; the row's bins cleared
__global__ __launch_bounds__(NT) void k_smp_stat(const float* logits, int n, SmpRow* rows) {
    __shared__ Shared sh;
    const int c = blockIdx.x, chunks = gridDim.x;
    SmpRow& r = rows[blockIdx.y];
    for (int b = c * NT + threadIdx.x; b < SMP_BINS; b += chunks * NT) r.mass[b] = 0, r.count[b] = 0;
    const Stat s = range_stat(logits + (size_t)blockIdx.y * n, chunk_begin(n, c, chunks), chunk_begin(n, c + 1, chunks), sh);
    if (threadIdx.x == 0) {
        r.first[c] = s.first;
        r.low[c] = s.low;
        r.nan[c] = s.nan;
        if (c == 0) r.n_list = 0;
    }
}

__device__ __forceinline__ Stat row_stat(const SmpRow& r, int chunks) {
    static_assert(SMP_CHUNKS == 64, "one chunk a lane");
    const int lane = threadIdx.x & 63;
    const bool in = lane < chunks;
    u64 first = in ? r.first[lane] : ~0ull;
    float low = in ? r.low[lane] : INFINITY;
    unsigned nan = in ? r.nan[lane] : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        first = min(first, shfl_xor64(first, o));
        low = fminf(low, __shfl_xor(low, o, 64));
        nan |= __shfl_xor(nan, o, 64);
    }
    return {first, low, nan != 0};
}

__global__ __launch_bounds__(NT) void k_smp_hist(const float* logits, int n, double one, double dead, SmpRules rules,
                                                 SmpRow* rows) {
    __shared__ Shared sh;
    const int c = blockIdx.x, chunks = gridDim.x;
    const gh_sampling rule = rules.r[blockIdx.y];
    SmpRow& r = rows[blockIdx.y];
    const Stat s = row_stat(r, chunks);
    if (s.nan || s.first == ~0ull || rule.temperature == 0.0f) return;
    const Weights w = weights_of(s, rule, one);
    clear_bins(sh);
    range_hist(logits + (size_t)blockIdx.y * n, chunk_begin(n, c, chunks), chunk_begin(n, c + 1, chunks), w,
               bins_of(s, w, dead), rule.top_k > 0, sh);
    for (int b = threadIdx.x; b < SMP_BINS; b += NT) {
        if (sh.mass[b]) atomicAdd(&r.mass[b], sh.mass[b]);
        if (sh.count[b]) atomicAdd(&r.count[b], sh.count[b]);
    }
}

__device__ __forceinline__ void load_bins(const SmpRow& r, Shared& sh) {
    for (int b = threadIdx.x; b < SMP_BINS; b += NT) sh.mass[b] = r.mass[b], sh.count[b] = r.count[b];
    __syncthreads();
}

__global__ __launch_bounds__(NT) void k_smp_gather(const float* logits, int n, double one, double dead, SmpRules rules,
                                                   SmpRow* rows) {
    __shared__ Shared sh;
    const int c = blockIdx.x, chunks = gridDim.x;
    const gh_sampling rule = rules.r[blockIdx.y];
    SmpRow& r = rows[blockIdx.y];
    const Stat s = row_stat(r, chunks);
    if (s.nan || s.first == ~0ull || rule.temperature == 0.0f) return;
    const Weights w = weights_of(s, rule, one);
    const Bins bins = bins_of(s, w, dead);
    load_bins(r, sh);
    const Cuts cuts = find_cuts(w, bins, rule, sh);
    range_gather(logits + (size_t)blockIdx.y * n, chunk_begin(n, c, chunks), chunk_begin(n, c + 1, chunks), bins, cuts,
                 r.list, &r.n_list);
}

__global__ __launch_bounds__(NT) void k_smp_pick(const float* logits, int n, double one, double dead, SmpRules rules,
                                                 const SmpRow* rows, int chunks, int32_t* tokens) {
    __shared__ Shared sh;
    const gh_sampling rule = rules.r[blockIdx.x];
    const SmpRow& r = rows[blockIdx.x];
    int32_t* token = tokens + blockIdx.x;
    const Stat s = row_stat(r, chunks);
    if (settled(s, rule, token)) return;
    const Weights w = weights_of(s, rule, one);
    const Bins bins = bins_of(s, w, dead);
    const unsigned listed = r.n_list;
    int t;
    if (listed <= SMP_LIST) {
        for (int i = threadIdx.x; i < (int)listed; i += NT) sh.list[i] = r.list[i];
        load_bins(r, sh);
        const Cuts cuts = find_cuts(w, bins, rule, sh);
        sort_list(sh, listed);
        t = pick(w, bins, rule, cuts, listed, sh);
    } else {
        t = slow_row(logits + (size_t)blockIdx.x * n, n, w, rule, sh);
    }
    if (threadIdx.x == 0) *token = t;
}

}  // namespace

int launch_sample_rows(const float* logits, int n_rows, int vocab, const SmpRules& rules, SmpRow* scratch, int32_t* tokens,
                       hipStream_t s) {
    const int bits = smp_bits(vocab);
    const double one = ldexp(1.0, bits), dead = (bits + 2) * 0.6931471805599453;
    const int chunks = smp_chunks(n_rows, vocab);
    if (chunks == 0) {
        hipLaunchKernelGGL(k_smp_row, dim3(n_rows), dim3(NT), 0, s, logits, vocab, one, dead, rules, tokens);
    } else {
        const dim3 grid(chunks, n_rows);
        hipLaunchKernelGGL(k_smp_stat, grid, dim3(NT), 0, s, logits, vocab, scratch);
        hipLaunchKernelGGL(k_smp_hist, grid, dim3(NT), 0, s, logits, vocab, one, dead, rules, scratch);
        hipLaunchKernelGGL(k_smp_gather, grid, dim3(NT), 0, s, logits, vocab, one, dead, rules, scratch);
        hipLaunchKernelGGL(k_smp_pick, dim3(n_rows), dim3(NT), 0, s, logits, vocab, one, dead, rules, (const SmpRow*)scratch,
                           chunks, tokens);
    }
    GH_HIP(hipGetLastError());
    return GH_OK;
}

}  // namespace gh
