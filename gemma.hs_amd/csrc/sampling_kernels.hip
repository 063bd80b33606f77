// gfx950 kernels of the batched sampler (temperature, top-k, top-p, min-p).
//
// The draw is a search along the ranks: for the top_k-th element, for the
// first whose running mass reaches top_p of what top_k left, for the first
// below min_p, and for the first whose running mass passes u times what the
// three leave.  None needs the row sorted:
//   1. largest and smallest logit, and the largest of each of some hundred
//      groups of the row (k_smp_stat);
//   2. (k_smp_hist) a row whose rules keep few elements, a short row: top_k
//      groups' largest are at least the top_k-th element, min_p is a fixed
//      distance from the largest: the elements that reach the nearer of the
//      two go straight to a list.  Any other row, a long one: a histogram over
//      SMP_BINS equal steps of the logit, with the number and the mass of each
//      bin's elements; running sums over the bins say in which bin, or few
//      bins, each search ends;
//   3. a long row's elements of those bins go to the list (k_smp_gather);
//   4. the list sorted, its running mass on top of the bins' in front of it:
//      the exact answers (k_smp_pick).
// A list that does not fit (rows with thousands of equal logits) is searched
// digit by digit instead (slow_row: 8 rows of 262144 equal logits 1.2 ms, 3
// with top_k and top_p).  Rows that one workgroup reads quickly run all steps
// in one kernel (k_smp_row).
//
// One row of 262144 logits with top_k is latency: 4.7, 6.4, 2.1 and 4.6 us for
// the four kernels, which a call's launches and its wait nearly hide.  64 rows
// of mixed rules: 15 us for k_smp_stat (67 MB at 4.4 TB/s), 18 for k_smp_hist
// (the weights' 64-bit arithmetic), 12 for k_smp_gather (those rows once more,
// from the last-level cache), 12.5 for k_smp_pick (one workgroup a row: the
// sort).  Five rows of 1024 by k_smp_row: 11.
#include <hip/hip_runtime.h>

#include "sampling.h"

namespace gh {

namespace {

typedef unsigned long long u64;
typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr double LOG2E = 1.44269504088896340736;

// Ascending in rank order: value descending, then index ascending.
__device__ __forceinline__ uint32_t value_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);  // -0 ranks as 0
    return (b & 0x80000000u) ? b : ~(b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k : ~k & 0x7fffffffu);
}
__device__ __forceinline__ u64 rank_key(float v, int i) { return ((u64)value_key(v) << 32) | (unsigned)i; }

// A row's weights exp((l - max) / T), as integers of `bits` fractional bits:
// their sums do not depend on the order, and are exact to 2^-bits a weight.
// In 64 bits because a draw compares sums over the whole vocabulary.
// 2^y = 2^k 2^f with |f| <= 1/2 and the series of exp(f ln 2) up to f^11, whose
// first term left out is below 2^-47; the sums' own steps are 2^-44 for 262144
// logits.  An infinite largest logit counts as 0, whose equals give y = inf,
// taken as 0; none of the others is asked for.
struct Weights {
    float top;
    double base;     // top, or 0 for an infinite one
    double log2e_t;  // log2(e) / T
    int bits;        // at most 51
    // (l - top) log2(e) / T must be above -1000
    __device__ __forceinline__ double scaled(float l, int e) const {
        constexpr double L = 0.693147180559945309417, L2 = L * L, L4 = L2 * L2, L8 = L4 * L4;
        const double y = fmin(((double)l - base) * log2e_t, 0.0), k = rint(y), f = y - k;
        double p = L8 * L2 * L / 39916800;
        p = fma(p, f, L8 * L2 / 3628800);
        p = fma(p, f, L8 * L / 362880);
        p = fma(p, f, L8 / 40320);
        p = fma(p, f, L4 * L2 * L / 5040);
        p = fma(p, f, L4 * L2 / 720);
        p = fma(p, f, L4 * L / 120);
        p = fma(p, f, L4 / 24);
        p = fma(p, f, L2 * L / 6);
        p = fma(p, f, L2 / 2);
        p = fma(p, f, L);
        p = fma(p, f, 1.0);
        return ldexp(p, (int)k + e);
    }
    __device__ __forceinline__ double real(float l) const { return scaled(l, 0); }
    // rounded by an addition: between 2^52 and 2^53 a double's low bits are the integer
    __device__ __forceinline__ u64 fixed(float l) const {
        return (u64)(__double_as_longlong(scaled(l, bits) + 0x1p52) - __double_as_longlong(0x1p52));
    }
};

// What the bins are: equal steps of top - l up to `reach`, behind which every
// weight is zero.  Monotonic in l, so that bins follow the ranks.  Half the
// distance, which no two finite logits take out of f32's range.  (An infinite
// top and its equals: a NaN, which is in reach and becomes bin 0.)
struct Bins {
    float half_top, scale, reach;  // bins a unit of half the distance; largest half the distance
    __device__ __forceinline__ float half(float l) const { return fmaf(-0.5f, l, half_top); }
    __device__ __forceinline__ bool in_reach(float l) const { return !(half(l) > reach); }
    __device__ __forceinline__ float place(float l) const { return half(l) * scale; }
    __device__ __forceinline__ int of(float l) const { return min((int)place(l), SMP_BINS - 1); }
};

// Values of other lanes without a trip through LDS, whose latency the chains of
// a sort or a sum would wait for at every step.  All lanes are active.
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ unsigned dpp(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, ROWS == 0xF);
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_XOR3 = 0x1B, DPP_XOR7 = 0x141, DPP_XOR8 = 0x128;
constexpr int DPP_UP = 0x110, DPP_ROW_LAST = 0x142, DPP_HALF_LAST = 0x143;

// v of lane ^ o; o a power of two below 64
__device__ __forceinline__ unsigned lane_xor(unsigned v, int o) {
    switch (o) {
        case 1: return dpp<DPP_XOR1>(v);
        case 2: return dpp<DPP_XOR2>(v);
        case 4: return dpp<DPP_XOR3>(dpp<DPP_XOR7>(v));
        case 8: return dpp<DPP_XOR8>(v);
        case 16: {
            const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
            return threadIdx.x & 16 ? r[0] : r[1];
        }
        default: {
            const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
            return threadIdx.x & 32 ? r[0] : r[1];
        }
    }
}
__device__ __forceinline__ u64 lane_xor(u64 v, int o) {
    const unsigned lo = lane_xor((unsigned)v, o), hi = lane_xor((unsigned)(v >> 32), o);
    return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ float lane_xor(float v, int o) { return __uint_as_float(lane_xor(__float_as_uint(v), o)); }

template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ u64 dpp(u64 v) {
    const unsigned lo = dpp<CTRL, ROWS>((unsigned)v), hi = dpp<CTRL, ROWS>((unsigned)(v >> 32));
    return ((u64)hi << 32) | lo;
}
// inclusive running sums over the wave's lanes
template <class T>
__device__ __forceinline__ T wave_scan(T v) {
    v += dpp<DPP_UP + 1>(v);
    v += dpp<DPP_UP + 2>(v);
    v += dpp<DPP_UP + 4>(v);
    v += dpp<DPP_UP + 8>(v);
    v += dpp<DPP_ROW_LAST, 0xA>(v);
    return v + dpp<DPP_HALF_LAST, 0xC>(v);
}

// LDS of a workgroup's reductions, of its bins, and of the list.
struct Small {
    u64 red[16];
    unsigned red32[16];
    float redf[16];
    int bin[8];
    u64 before[8], upto[8];
    unsigned n_list;
};
struct BinSums {
    u64 mass[SMP_BINS];  // per bin, then running
    unsigned count[SMP_BINS];
};

template <int NT, class Op>
__device__ __forceinline__ u64 block_reduce(u64 v, Small& sh, Op op) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = op(v, lane_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh.red[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) v = op(v, sh.red[i]);
    return v;
}

// inclusive running sums over the threads
template <int NT>
__device__ __forceinline__ void block_scan(u64& m, unsigned& c, Small& sh) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    m = wave_scan(m);
    c = wave_scan(c);
    __syncthreads();
    if (lane == 63) sh.red[w] = m, sh.red32[w] = c;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i)
        if (i < w) m += sh.red[i], c += sh.red32[i];
}

// The distance from the largest logit at which a weight, below 2^-(bits + 2),
// rounds to zero; as f32 no shorter than it is.
__device__ __forceinline__ double dead_of(int bits, double log2e_t) { return (bits + 2) / log2e_t; }
__device__ __forceinline__ float dead_of(int bits, float temperature) {
    return (float)(dead_of(bits, LOG2E / (double)temperature) * 1.000001);
}

// ------------------------------------------------------------------
// step 1
// ------------------------------------------------------------------
struct Stat {
    u64 first;  // rank key of the first in rank order; ~0: nothing above -inf
    float low;  // smallest of those that may have a weight, or one below it
    bool nan;
    float own;  // the largest of the elements that this thread read
};

// The elements [i0, i1) of a row (l is aligned to 4) as 16-byte quads between
// the first and the last 16-byte boundary, and up to 6 elements at the edges.
struct Quads {
    const f32x4* p;
    int first, quads, i0, head, i1, tail;
    __device__ __forceinline__ Quads(const float* l, int i0, int i1) : i0(i0), i1(i1) {
        head = min((int)(-((uintptr_t)(l + i0) >> 2) & 3), i1 - i0);
        first = i0 + head;
        quads = (i1 - first) / 4;
        tail = i1 - first - 4 * quads;
        p = (const f32x4*)(l + first);
    }
    // index of the thread's element at the edges, or -1
    __device__ __forceinline__ int edge(int tid) const {
        return tid < head ? i0 + tid : tid < head + tail ? i1 - tail + tid - head : -1;
    }
};

// f(index, logit) of the elements [i0, i1), U loads in flight a thread
template <int NT, int U, class F>
__device__ __forceinline__ void each_logit(const float* l, int i0, int i1, F&& f) {
    const Quads r(l, i0, i1);
#pragma unroll 1
    for (int q = threadIdx.x; q < r.quads; q += U * NT) {
        f32x4 v[U];
#pragma unroll
        for (int j = 0; j < U; ++j) v[j] = r.p[min(q + j * NT, r.quads - 1)];
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (q + j * NT < r.quads) {
#pragma unroll
                for (int e = 0; e < 4; ++e) f(r.first + 4 * (q + j * NT) + e, v[j][e]);
            }
    }
    if (const int i = r.edge(threadIdx.x); i >= 0) f(i, l[i]);
}

// largest over 16 lanes
__device__ __forceinline__ float max16(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, lane_xor(v, o));
    return v;
}

// dead: the distance from the largest at which a weight is zero.  Masked
// logits, of the type's lowest value or the like, have to stay out of `low`:
// bins that reached so far would be few for the others.  What is that far
// below the largest of the first 256 that 16 lanes read is that far below the
// row's.
template <int NT>
__device__ __forceinline__ Stat range_stat(const float* l, int i0, int i1, float dead, Small& sh) {
    constexpr int U = 4;
    const Quads r(l, i0, i1);
    float best = -INFINITY, low = INFINITY;
    int at = -1;  // index of the best, or of the first of its quad
    float floor = -3.4028234e38f;
    bool nan = false;
    auto one = [&](int i, float v) {
        nan |= v != v;
        if (v > best || (v == best && i < at)) best = v, at = i;
        low = fminf(low, v >= floor ? v : INFINITY);
    };
#pragma unroll 1
    for (int q = threadIdx.x; q < r.quads; q += U * NT) {
        f32x4 v[U];
#pragma unroll
        for (int j = 0; j < U; ++j) v[j] = r.p[min(q + j * NT, r.quads - 1)];
        if (q == (int)threadIdx.x) {
            float m = -INFINITY;
#pragma unroll
            for (int j = 0; j < U; ++j) m = fmaxf(m, fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(v[j].z, v[j].w)));
            floor = fmaxf(floor, max16(m) - dead);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            // The last quad may come more than once: not for `best`, which is
            // also the largest of this thread's elements alone.  A thread's
            // quads ascend, so that the first of equal ones stays.
            const float hi = q + j * NT < r.quads ? fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(v[j].z, v[j].w)) : -INFINITY;
            float lo = fminf(fminf(v[j].x, v[j].y), fminf(v[j].z, v[j].w));
            nan |= __builtin_isunordered(v[j].x, v[j].y) | __builtin_isunordered(v[j].z, v[j].w);
            if (hi > best) best = hi, at = r.first + 4 * (q + j * NT);
            if (lo < floor) {
                lo = INFINITY;
#pragma unroll
                for (int e = 0; e < 4; ++e) lo = fminf(lo, v[j][e] >= floor ? v[j][e] : INFINITY);
            }
            low = fminf(low, lo);
        }
    }
    if (at >= 0) {  // which of the quad
        const f32x4 v = r.p[(at - r.first) / 4];
        at += v.x == best ? 0 : v.y == best ? 1 : v.z == best ? 2 : 3;
    }
    if (const int i = r.edge(threadIdx.x); i >= 0) one(i, l[i]);
    u64 first = at >= 0 ? rank_key(best, at) : ~0ull;
    unsigned bad = __any(nan);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        first = min(first, lane_xor(first, o));
        low = fminf(low, lane_xor(low, o));
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        sh.red[threadIdx.x >> 6] = first;
        sh.redf[threadIdx.x >> 6] = low;
        sh.red32[threadIdx.x >> 6] = bad;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        first = min(first, sh.red[i]);
        low = fminf(low, sh.redf[i]);
        bad |= sh.red32[i];
    }
    return {first, low, bad != 0, best};
}

// the row is drawn from: no NaN, something above -inf, and not greedy
__device__ __forceinline__ bool drawn(const Stat& s, const gh_sampling& rule) {
    return !s.nan && s.first != ~0ull && rule.temperature > 0.0f;
}
__device__ __forceinline__ int token_of_undrawn(const Stat& s) { return s.nan || s.first == ~0ull ? -1 : (int)(unsigned)s.first; }

__device__ __forceinline__ Weights weights_of(const Stat& s, const gh_sampling& rule, int bits) {
    const float top = key_value((unsigned)(s.first >> 32));
    return {top, top == INFINITY ? 0.0 : (double)top, LOG2E / (double)rule.temperature, bits};
}

__device__ __forceinline__ Bins bins_of(const Stat& s, const Weights& w) {
    const double dead = dead_of(w.bits, w.log2e_t), span = (double)w.top - (double)s.low, d = span < dead ? span : dead;
    if (!(d > 0.0)) return {0.5f * w.top, 0.0f, 0.0f};  // one value: one bin
    return {0.5f * w.top, (float)fmin(2.0 * SMP_BINS / d, 3e38), (float)fmin(d * 0.5000005, 3.4028234e38)};
}

// ------------------------------------------------------------------
// step 2
// ------------------------------------------------------------------
template <int NT>
__device__ __forceinline__ void clear_bins(BinSums& h) {
    for (int b = threadIdx.x; b < SMP_BINS; b += NT) h.mass[b] = 0, h.count[b] = 0;
    __syncthreads();
}

template <int NT>
__device__ __forceinline__ void range_hist(const float* l, int i0, int i1, const Weights& w, const Bins& bins, bool counts,
                                           BinSums& h) {
    clear_bins<NT>(h);
    each_logit<NT, 2>(l, i0, i1, [&](int, float v) {
        if (!bins.in_reach(v)) return;
        const u64 m = w.fixed(v);
        const int b = bins.of(v);
        if (m) {
            atomicAdd(&h.mass[b], m);
            if (counts) atomicAdd(&h.count[b], 1u);
        }
    });
    __syncthreads();
}

// ------------------------------------------------------------------
// step 3: where the searches end, from the bins alone
// ------------------------------------------------------------------
// Running sums over the bins, a thread's own ones in its registers: m[j], c[j]
// in front of bin b0 + j.
template <int NT>
struct Running {
    static constexpr int PER = SMP_BINS / NT;
    u64 m[PER + 1];
    unsigned c[PER + 1];
    int b0;
    __device__ __forceinline__ Running(const u64* mass, const unsigned* count, Small& sh) : b0(threadIdx.x * PER) {
        u64 sum = 0;
        unsigned csum = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            m[j + 1] = mass[b0 + j];
            c[j + 1] = count[b0 + j];
            sum += m[j + 1];
            csum += c[j + 1];
        }
        u64 run = sum;
        unsigned crun = csum;
        block_scan<NT>(run, crun, sh);
        m[0] = run - sum;
        c[0] = crun - csum;
#pragma unroll
        for (int j = 0; j < PER; ++j) m[j + 1] += m[j], c[j + 1] += c[j];
        if (threadIdx.x == NT - 1) sh.upto[7] = m[PER], sh.bin[6] = (int)c[PER];  // of all
    }
    // The bin in which a running sum first satisfies `reached` (false for 0):
    // slot i of sh.
    template <class P>
    __device__ __forceinline__ void find(int i, Small& sh, P&& reached) const {
        bool there = reached(m[0], c[0]);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const bool here = reached(m[j + 1], c[j + 1]);
            if (here && !there) put(i, j, sh);
            there = here;
        }
    }
    __device__ __forceinline__ void put(int i, int j, Small& sh) const {
        sh.bin[i] = b0 + j;
        sh.before[i] = m[j];
        sh.upto[i] = m[j + 1];
    }
    // bin b as slot i
    __device__ __forceinline__ void look(int i, int b, Small& sh) const {
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (b0 + j == b) put(i, j, sh);
    }
    // the sums up to and with each bin
    __device__ __forceinline__ void store(u64* mass, unsigned* count) const {
#pragma unroll
        for (int j = 0; j < PER; ++j) mass[b0 + j] = m[j + 1], count[b0 + j] = c[j + 1];
    }
};

// Where in the bins a weight falls below min_p, to be taken with a bin to
// either side for roundings.
__device__ __forceinline__ double min_p_bin(const Weights& w, const Bins& bins, const gh_sampling& rule) {
    return (double)-log2f(rule.min_p) / w.log2e_t * 0.5 * (double)bins.scale;
}

template <int NT>
__device__ __forceinline__ SmpCuts find_cuts(const Weights& w, const Bins& bins, const gh_sampling& rule, const Running<NT>& run,
                                             Small& sh) {
    __syncthreads();
    SmpCuts q;
    q.total = sh.upto[7];
    // what is behind the last element with a weight cannot be drawn: a top_k
    // that reaches there leaves all the mass
    q.k = rule.top_k > 0 && rule.top_k < sh.bin[6];
    q.p = rule.top_p < 1.0f;
    const double d = rule.min_p > 0.0f ? min_p_bin(w, bins, rule) : SMP_BINS + 1;
    q.m = d < SMP_BINS + 1;  // else every weight reaches it
    for (int i = 0; i < 4; ++i) q.lo[i] = 1, q.hi[i] = 0;
    if (q.k) {
        const unsigned k = rule.top_k;
        run.find(0, sh, [&](u64, unsigned c) { return c >= k; });
    }
    if (q.m) {
        q.lo[2] = max((int)d - 1, 0);
        q.hi[2] = min((int)d + 1, SMP_BINS - 1);
        run.look(1, q.lo[2], sh);
        run.look(2, q.hi[2], sh);
    }
    if (q.k || q.m) __syncthreads();
    u64 zlo = q.total, zhi = q.total;  // mass that top_k leaves
    if (q.k) {
        q.lo[0] = q.hi[0] = sh.bin[0];
        zlo = sh.before[0];
        zhi = sh.upto[0];
    }
    u64 lo = zlo, hi = zhi;  // mass that all three leave
    q.upto_m = q.total;
    if (q.m) {
        q.upto_m = sh.upto[2];
        lo = min(lo, sh.before[1]);
        hi = min(hi, q.upto_m);
    }
    if (q.p) {
        const double tlo = (double)rule.top_p * (double)zlo, thi = (double)rule.top_p * (double)zhi;
        run.find(3, sh, [&](u64 m, unsigned) { return m > 0 && (double)m >= tlo; });
        run.find(4, sh, [&](u64 m, unsigned) { return m > 0 && (double)m >= thi; });
        __syncthreads();
        q.lo[1] = sh.bin[3];
        q.hi[1] = sh.bin[4];
        lo = min(lo, sh.before[3]);
        hi = min(hi, sh.upto[4]);
    }
    const double ulo = (double)rule.u * (double)lo, uhi = (double)rule.u * (double)hi;
    run.find(5, sh, [&](u64 m, unsigned) { return (double)m > ulo; });
    run.find(7, sh, [&](u64 m, unsigned) { return (double)m > uhi; });
    __syncthreads();
    q.lo[3] = sh.bin[5];
    q.hi[3] = sh.bin[7];
    __syncthreads();
    return q;
}

// To the list, n elements of it taken: the elements of the bins [lo, hi] that
// `in` takes.  They meet in LDS (`near`, SMP_BINS of them; sh.n_list 0 before)
// and go out together: an atomic on the row's own counter for each would hold
// its wave for a round trip.
template <int NT, class In>
__device__ __forceinline__ void range_gather(const float* l, int i0, int i1, const Bins& bins, int lo, int hi, u64* list,
                                             unsigned* n, u64* near, Small& sh, In&& in) {
    const float from = (float)lo, to = hi < SMP_BINS - 1 ? (float)(hi + 1) : INFINITY;
    each_logit<NT, 4>(l, i0, i1, [&](int i, float v) {
        // most elements are none of them, and are known by one product
        const float t = bins.place(v);
        if (t < from || t >= to) return;
        if (!bins.in_reach(v)) return;
        const int b = bins.of(v);
        if (b < lo || b > hi || !in(b)) return;
        unsigned at = atomicAdd(&sh.n_list, 1u);
        if (at < SMP_BINS) {
            near[at] = rank_key(v, i);
        } else {
            at = atomicAdd(n, 1u);
            if (at < SMP_LIST) list[at] = rank_key(v, i);
        }
    });
    __syncthreads();
    const unsigned count = min(sh.n_list, (unsigned)SMP_BINS);
    if (threadIdx.x == 0 && count) sh.bin[7] = (int)atomicAdd(n, count);
    __syncthreads();
    const unsigned first = sh.bin[7];
    for (unsigned i = threadIdx.x; i < count; i += NT)
        if (first + i < SMP_LIST) list[first + i] = near[i];
}
template <int NT>
__device__ __forceinline__ void range_gather(const float* l, int i0, int i1, const Bins& bins, const SmpCuts& q, u64* list,
                                             unsigned* n, u64* near, Small& sh) {
    int lo = SMP_BINS, hi = -1;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (q.lo[j] <= q.hi[j]) lo = min(lo, q.lo[j]), hi = max(hi, q.hi[j]);
    range_gather<NT>(l, i0, i1, bins, lo, hi, list, n, near, sh, [&](int b) {
        bool in = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) in |= b >= q.lo[j] && b <= q.hi[j];
        return in;
    });
}

// Counts per bin become running counts.
template <int NT>
__device__ __forceinline__ void scan_counts(unsigned* count, Small& sh) {
    constexpr int PER = SMP_BINS / NT;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, b0 = threadIdx.x * PER;
    unsigned c[PER], sum = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += c[j] = count[b0 + j];
    unsigned run = wave_scan(sum);
    if (lane == 63) sh.red32[w] = run;
    __syncthreads();
    run -= sum;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i)
        if (i < w) run += sh.red32[i];
#pragma unroll
    for (int j = 0; j < PER; ++j) count[b0 + j] = run += c[j];
    __syncthreads();
}

// A short row: the last bin of the elements that its list needs (-1: a long
// row), and whether top_p needs the mass of all (the list has what top_k
// leaves).  top_k: the bin in which the groups' largest come to top_k; where
// top_p asks for the mass that top_k leaves, min_p must not cut the list.  A
// row is short if at most half of its groups reach that far: about as many
// elements do.
struct Short {
    int last;
    bool all;
};
template <int NT>
__device__ __forceinline__ Short short_row(const float* group_max, int groups, const Weights& w, const Bins& bins,
                                           const gh_sampling& rule, BinSums& h, Small& sh) {
    const bool k = rule.top_k > 0 && rule.top_k <= groups / 2;
    const bool m = rule.min_p > 0.0f && (rule.top_p >= 1.0f || rule.top_k == 0);
    if (!k && !m) return {-1, false};
    for (int b = threadIdx.x; b < SMP_BINS; b += NT) h.count[b] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < groups; i += NT) {
        const float v = group_max[i];
        if (bins.in_reach(v)) atomicAdd(&h.count[bins.of(v)], 1u);
    }
    __syncthreads();
    scan_counts<NT>(h.count, sh);
    int last = SMP_BINS - 1;
    if (k && h.count[SMP_BINS - 1] >= (unsigned)rule.top_k) {
        for (int b = threadIdx.x; b < SMP_BINS; b += NT)
            if (h.count[b] >= (unsigned)rule.top_k && (b == 0 || h.count[b - 1] < (unsigned)rule.top_k)) sh.bin[0] = b;
        __syncthreads();
        last = sh.bin[0];
    }
    if (m) last = min(last, (int)fmin(min_p_bin(w, bins, rule) + 1.0, (double)(SMP_BINS - 1)));
    const bool is_short = h.count[last] <= (unsigned)groups / 2;
    __syncthreads();
    return {is_short ? last : -1, rule.top_p < 1.0f && rule.top_k == 0};
}

// Mass of the elements [i0, i1); in every thread.
template <int NT>
__device__ __forceinline__ u64 range_mass(const float* l, int i0, int i1, const Weights& w, const Bins& bins, Small& sh) {
    u64 sum = 0;
    each_logit<NT, 2>(l, i0, i1, [&](int, float v) {
        if (bins.in_reach(v)) sum += w.fixed(v);
    });
    return block_reduce<NT>(sum, sh, [](u64 a, u64 b) { return a + b; });
}

// ------------------------------------------------------------------
// step 4, 1024 threads
// ------------------------------------------------------------------
constexpr int PT = 1024;

struct PickShared {
    u64 list[SMP_LIST];
    u64 upto[PT];  // running mass of a thread's last element
    u64 off_mass[SMP_LIST];
    unsigned off_count[SMP_LIST];
    u64 found[4];
    u64 mass_at[4];
    int at[4];
};

// One merge of a bitonic sort within the wave's lanes: runs of k elements
// around `at`, the distances of a half run and less.
__device__ __forceinline__ void merge_lanes(u64& x, int k, int at) {
#pragma unroll
    for (int j = 32; j > 0; j >>= 1) {
        if (j >= k) continue;
        const u64 y = lane_xor(x, j);
        const bool up = (at & k) == 0, lower = (at & j) == 0;
        x = (x < y) == (up == lower) ? x : y;
    }
}

// ascending, in LDS; n <= PER * PT.  A thread holds PER elements PT apart, so
// that only the distances from 64 to PT / 2 pass through LDS.
template <int PER>
__device__ __forceinline__ void sort_list(u64* list, int n) {
    const int tid = threadIdx.x;
    int size = PER > 1 ? PER * PT : 64;
    while (size < n) size *= 2;
    u64 x[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) x[e] = tid + e * PT < n ? list[tid + e * PT] : ~0ull;
    for (int k = 2; k <= size; k *= 2) {
        int j = k / 2;
#pragma unroll
        for (int half = PER / 2; half > 0; half /= 2) {
            if (j < half * PT) continue;
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                if (e & half) continue;
                const bool up = ((tid + e * PT) & k) == 0;
                const u64 lo = min(x[e], x[e + half]), hi = max(x[e], x[e + half]);
                x[e] = up ? lo : hi;
                x[e + half] = up ? hi : lo;
            }
            j = half * PT / 2;
        }
        for (; j >= 64; j /= 2) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < PER; ++e)
                if (PER > 1 || tid < size) list[tid + e * PT] = x[e];
            __syncthreads();
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const int i = tid + e * PT;
                const u64 y = PER > 1 || tid < size ? list[i ^ j] : ~0ull;
                const bool up = (i & k) == 0, lower = (i & j) == 0;
                x[e] = (x[e] < y) == (up == lower) ? x[e] : y;
            }
        }
#pragma unroll
        for (int e = 0; e < PER; ++e) merge_lanes(x[e], k, tid + e * PT);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; ++e)
        if (PER > 1 || tid < size) list[tid + e * PT] = x[e];
    __syncthreads();
}

// The token, from the list and the running sums of the bins in front
// of its elements (LDS or global; none for a list that begins with the row's
// first element and leaves none out), PER elements a thread.
template <int PER>
__device__ __forceinline__ int pick(const Weights& w, const Bins& bins, const gh_sampling& rule, const SmpCuts& cuts,
                                    const u64* mass, const unsigned* count, int n, PickShared& p, Small& sh) {
    sort_list<PER>(p.list, n);
    auto bin_of = [&](float v) { return mass ? bins.of(v) : 0; };
    const int tid = threadIdx.x;
    u64 upto[PER];       // running mass up to and with the element
    unsigned rank[PER];  // and its rank, from 1
    float val[PER];
    u64 m[PER];
    {
        u64 s = 0;
        int b[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = tid * PER + j;
            val[j] = i < n ? key_value((unsigned)(p.list[i] >> 32)) : 0.0f;
            m[j] = i < n ? w.fixed(val[j]) : 0;
            b[j] = i < n ? bin_of(val[j]) : -1;
            s += m[j];
        }
        u64 at = s;
        unsigned none = 0;
        block_scan<PT>(at, none, sh);
        at -= s;  // of the list in front of this thread
        // What the elements' running sums in the list lack, of each bin of it:
        // written by the bin's first element for those behind it (the bins
        // are at most as many as the elements; p.off_* by the first's place).
        int prev = tid * PER > 0 && tid * PER <= n ? bin_of(key_value((unsigned)(p.list[tid * PER - 1] >> 32))) : -1;
        int head[PER];  // place of the first element of the bin, if it is one of this thread's, else -1
        u64 run = at;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = tid * PER + j;
            const bool first = i < n && b[j] != prev;
            head[j] = first ? i : -1;
            if (first) {
                p.off_mass[i] = (b[j] > 0 ? mass[b[j] - 1] : 0) - run;
                p.off_count[i] = (b[j] > 0 ? count[b[j] - 1] : 0) - i;
            }
            run += m[j];
            prev = b[j];
        }
        // place of the first element of each element's bin: running maximum of the heads
        int h = -1;
#pragma unroll
        for (int j = 0; j < PER; ++j) h = max(h, head[j]);
        int inc = h;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(inc, o, 64);
            if ((tid & 63) >= o) inc = max(inc, y);
        }
        __syncthreads();
        if ((tid & 63) == 63) sh.red32[tid >> 6] = (unsigned)(inc + 1);
        __syncthreads();
        int before = __shfl_up(inc, 1, 64);
        if ((tid & 63) == 0) before = -1;
#pragma unroll
        for (int i = 0; i < PT / 64; ++i)
            if (i < tid >> 6) before = max(before, (int)sh.red32[i] - 1);
        run = at;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = tid * PER + j;
            if (head[j] >= 0) before = head[j];
            run += m[j];
            upto[j] = i < n ? p.off_mass[before] + run : 0;
            rank[j] = i < n ? p.off_count[before] + i + 1 : 0;
        }
    }
    p.upto[tid] = upto[PER - 1];
    if (tid < 4) p.at[tid] = n;
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (tid * PER + j == n - 1) p.found[0] = p.found[1] = upto[j];  // a search that ends behind the list: all of it
    __syncthreads();
    // `reached`, false and then true along the list: p.at[slot] the place of
    // the first true, p.found[slot] its running mass
    auto first = [&](int slot, auto&& reached) {
        bool before = tid > 0 && tid * PER <= n && reached(-1);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = tid * PER + j;
            const bool here = i < n && reached(j);
            if (here && !before) {
                p.at[slot] = i;
                p.found[slot] = upto[j];
                p.mass_at[slot] = m[j];
            }
            before = here;
        }
        __syncthreads();
    };
    auto of = [&](int j) { return j < 0 ? p.upto[tid - 1] : upto[j]; };
    u64 left = cuts.total ? cuts.total : p.found[0], most = mass ? cuts.upto_m : p.found[0];
    u64 kept = min(left, p.found[0] | (mass ? ~0ull : 0));
    if (cuts.k) {
        __syncthreads();
        // ranks of the elements without a weight may repeat; they are the last
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (tid * PER + j < n && rank[j] == (unsigned)rule.top_k && m[j]) p.found[0] = upto[j];
        __syncthreads();
        left = kept = p.found[0];
    }
    if (cuts.p) {
        const double t = (double)rule.top_p * (double)left;
        first(1, [&](int j) { return (double)of(j) >= t; });
        kept = min(kept, p.found[1]);
    }
    if (cuts.m) {
        const double t = (double)rule.min_p;
        first(2, [&](int j) {
            return w.real(j < 0 ? key_value((unsigned)(p.list[tid * PER - 1] >> 32)) : val[j]) < t;
        });
        kept = min(kept, most);
        if (p.at[2] < n) kept = min(kept, p.found[2] - p.mass_at[2]);
    }
    const double t = (double)rule.u * (double)kept;
    first(3, [&](int j) { return (double)of(j) > t; });
    return (int)(unsigned)p.list[p.at[3]];
}

// The same for a list of at most 64 by one wave alone: no barriers, and little
// code, which the first passes of a kernel have to fetch.
__device__ __forceinline__ int pick_wave(const Weights& w, const Bins& bins, const gh_sampling& rule, const SmpCuts& cuts,
                                         const u64* mass, const unsigned* count, u64 key, int n) {
    const int lane = threadIdx.x & 63;
    if (lane >= n) key = ~0ull;
#pragma unroll 1
    for (int k = 2; k <= 64; k *= 2) merge_lanes(key, k, lane);
    const bool in = lane < n;
    const float val = in ? key_value((unsigned)(key >> 32)) : 0.0f;
    const double real = in ? w.real(val) : 0.0;
    const u64 m = in ? w.fixed(val) : 0;
    u64 upto = wave_scan(m);
    const u64 listed = ((u64)(unsigned)__shfl((int)(upto >> 32), 63, 64) << 32) | (unsigned)__shfl((int)upto, 63, 64);
    int rank = lane + 1;
    if (mass) {  // on top of the bins in front: what the bin's first element lacks, for those behind it too
        const int b = in ? bins.of(val) : -1, prev = __shfl_up(b, 1, 64);
        const bool head = in && (lane == 0 || b != prev);
        const u64 off = head ? (b > 0 ? mass[b - 1] : 0) - (upto - m) : 0;
        const int off_rank = head ? (b > 0 ? (int)count[b - 1] : 0) - lane : 0;
        const u64 heads = __ballot(head) & (~0ull >> (63 - lane));
        const int from = 63 - __clzll((long long)(heads | 1));
        upto += ((u64)(unsigned)__shfl((int)(off >> 32), from, 64) << 32) | (unsigned)__shfl((int)off, from, 64);
        rank += __shfl(off_rank, from, 64);
    }
    auto at = [&](u64 v, u64 lanes, u64 none) {  // v of the first of the lanes
        if (!lanes) return none;
        const int from = __ffsll((long long)lanes) - 1;
        return ((u64)(unsigned)__shfl((int)(v >> 32), from, 64) << 32) | (unsigned)__shfl((int)v, from, 64);
    };
    u64 left = cuts.total ? cuts.total : listed, kept = mass ? left : min(left, listed);
    if (cuts.k) left = kept = at(upto, __ballot(in && m && rank == rule.top_k), listed);
    if (cuts.p) {
        const double t = (double)rule.top_p * (double)left;
        kept = min(kept, at(upto, __ballot(in && (double)upto >= t), listed));
    }
    if (cuts.m) {
        if (mass) kept = min(kept, cuts.upto_m);
        kept = min(kept, at(upto - m, __ballot(in && real < (double)rule.min_p), kept));
    }
    const double t = (double)rule.u * (double)kept;
    return (int)(unsigned)at(key, __ballot(in && (double)upto > t), 0);
}

// ------------------------------------------------------------------
// rows whose list is too long, 1024 threads
// ------------------------------------------------------------------
struct SlowShared {
    u64 mass[256];
    unsigned count[256];
    u64 key, base_mass;
    unsigned base_count;
};

// The first element in rank order whose running count reaches `k` (k > 0), or
// whose running mass reaches (strict: passes) `t`: digit by digit of its rank
// key, from the counts and masses of the 256 values of each digit among the
// elements that share the digits before.  The mass up to and with it goes to
// sh.base_mass, its key to sh.key.
__device__ void find(const float* l, int n, const Weights& w, const Bins& bins, unsigned k, double t, bool strict, SlowShared& sh) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid == 0) sh.key = sh.base_mass = 0, sh.base_count = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        if (shift == 24) continue;  // indexes are below 2^24
        if (tid < 256) sh.mass[tid] = 0, sh.count[tid] = 0;
        __syncthreads();
        const u64 prefix = sh.key;
        // equal logits are what brings rows here: a thread's equal digits in a
        // row go out together (8 rows of 262144 in 1.2 ms, one by one 2.8)
        int last = 0;
        u64 mass = 0;
        unsigned count = 0;
        auto out = [&] {
            if (count) atomicAdd(&sh.count[last], count);
            if (mass) atomicAdd(&sh.mass[last], mass);
        };
        each_logit<PT, 2>(l, 0, n, [&](int i, float v) {
            const u64 key = rank_key(v, i);
            if (shift < 56 && (key >> (shift + 8)) != (prefix >> (shift + 8))) return;
            const int d = (int)(key >> shift) & 255;
            if (d != last) {
                out();
                last = d;
                mass = count = 0;
            }
            ++count;
            if (bins.in_reach(v)) mass += w.fixed(v);
        });
        out();
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
    if (tid == 0 && bins.in_reach(l[(unsigned)sh.key])) sh.base_mass += w.fixed(l[(unsigned)sh.key]);
    __syncthreads();
}

__device__ __noinline__ int slow_row(const float* l, int n, const Weights& w, const Bins& bins, const gh_sampling& rule, SlowShared& sh, Small& red) {
    u64 total = 0, at_least = 0;
    each_logit<PT, 2>(l, 0, n, [&](int, float v) {
        if (!bins.in_reach(v)) return;
        const u64 m = w.fixed(v);
        total += m;
        if (w.real(v) >= (double)rule.min_p) at_least += m;
    });
    auto plus = [](u64 a, u64 b) { return a + b; };
    total = block_reduce<PT>(total, red, plus);
    at_least = block_reduce<PT>(at_least, red, plus);
    if (rule.top_k > 0 && rule.top_k < n) {
        find(l, n, w, bins, rule.top_k, 0.0, false, sh);
        total = sh.base_mass;
    }
    u64 kept = min(total, at_least);
    if (rule.top_p < 1.0f) {
        find(l, n, w, bins, 0, (double)rule.top_p * (double)total, false, sh);
        kept = min(kept, sh.base_mass);
    }
    find(l, n, w, bins, 0, (double)rule.u * (double)kept, true, sh);
    return (int)(unsigned)sh.key;
}

// ------------------------------------------------------------------
// kernels
// ------------------------------------------------------------------
// Rules of a short row; total 0: its list has all the mass.
__device__ __forceinline__ SmpCuts short_cuts(const gh_sampling& rule, u64 total) {
    SmpCuts q;
    q.total = total;
    q.k = rule.top_k > 0;
    q.p = rule.top_p < 1.0f;
    q.m = rule.min_p > 0.0f;
    return q;
}

// one workgroup a row
__global__ __launch_bounds__(PT) void k_smp_row(const float* logits, int n, int bits, SmpRules rules, int32_t* tokens) {
    __shared__ Small sh;
    __shared__ BinSums h;
    __shared__ union {
        PickShared p;
        SlowShared slow;
        float group_max[PT];
    } u;
    __shared__ u64 near[SMP_BINS];
    __shared__ unsigned listed_row;
    const SmpRule rule = rules.r[blockIdx.x];
    const int at = rule.row;
    const float* l = logits + (size_t)at * n;
    const int tid = threadIdx.x;
    const Stat s = range_stat<PT>(l, 0, n, dead_of(bits, rule.temperature), sh);
    if (!drawn(s, rule)) {
        if (tid == 0) tokens[at] = token_of_undrawn(s);
        return;
    }
    const Weights w = weights_of(s, rule, bits);
    const Bins bins = bins_of(s, w);
    u.group_max[tid] = s.own;
    if (tid == 0) sh.n_list = listed_row = 0;
    __syncthreads();
    const Short row = short_row<PT>(u.group_max, PT, w, bins, rule, h, sh);
    SmpCuts cuts;
    const bool is_short = row.last >= 0;
    if (is_short) {
        cuts = short_cuts(rule, row.all ? range_mass<PT>(l, 0, n, w, bins, sh) : 0);
        range_gather<PT>(l, 0, n, bins, 0, row.last, u.p.list, &listed_row, near, sh, [](int) { return true; });
    } else {
        range_hist<PT>(l, 0, n, w, bins, rule.top_k > 0, h);
        const Running<PT> run(h.mass, h.count, sh);
        cuts = find_cuts<PT>(w, bins, rule, run, sh);
        run.store(h.mass, h.count);
        range_gather<PT>(l, 0, n, bins, cuts, u.p.list, &listed_row, near, sh);
    }
    __syncthreads();
    const unsigned listed = listed_row;
    const u64* mass = is_short ? nullptr : h.mass;
    int t;
    if (listed <= 64) {
        if (tid >= 64) return;
        t = pick_wave(w, bins, rule, cuts, mass, h.count, u.p.list[tid], listed);
    } else if (listed <= SMP_LIST) {
        t = listed <= PT ? pick<1>(w, bins, rule, cuts, mass, h.count, listed, u.p, sh)
                         : pick<SMP_LIST / PT>(w, bins, rule, cuts, mass, h.count, listed, u.p, sh);
    } else {
        t = slow_row(l, n, w, bins, rule, u.slow, sh);
    }
    if (tid == 0) tokens[at] = t;
}

__device__ __forceinline__ int chunk_begin(int n, int c, int chunks) { return (int)((int64_t)n * c / chunks); }

constexpr int CT = 512;  // threads of a workgroup that reads a chunk of a row

// a row's chunks: stats; the row's bins cleared
__global__ __launch_bounds__(CT) void k_smp_stat(const float* logits, int n, int bits, int group, SmpRules rules, SmpRow* rows) {
    __shared__ Small sh;
    const int c = blockIdx.x, chunks = gridDim.x, tid = threadIdx.x;
    SmpRow& r = rows[blockIdx.y];
    for (int b = c * CT + tid; b < SMP_BINS; b += chunks * CT) r.mass[b] = 0, r.count[b] = 0;
    const SmpRule rule = rules.r[blockIdx.y];
    const Stat s = range_stat<CT>(logits + (size_t)rule.row * n, chunk_begin(n, c, chunks), chunk_begin(n, c + 1, chunks),
                                  dead_of(bits, rule.temperature), sh);
    float own = s.own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
        if (o < group) own = fmaxf(own, lane_xor(own, o));
    if (tid % group == 0) r.group_max[(c * CT + tid) / group] = own;
    if (tid == 0) {
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
    const bool nan = __any(in && r.nan[lane]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        first = min(first, lane_xor(first, o));
        low = fminf(low, lane_xor(low, o));
    }
    return {first, low, nan, 0.0f};
}

// A short row: its list.  A long one: its bins.
__global__ __launch_bounds__(CT) void k_smp_hist(const float* logits, int n, int bits, int groups, SmpRules rules, SmpRow* rows) {
    __shared__ Small sh;
    __shared__ BinSums h;
    const int c = blockIdx.x, chunks = gridDim.x, tid = threadIdx.x;
    const SmpRule rule = rules.r[blockIdx.y];
    SmpRow& r = rows[blockIdx.y];
    const Stat s = row_stat(r, chunks);
    if (!drawn(s, rule)) return;
    const Weights w = weights_of(s, rule, bits);
    const Bins bins = bins_of(s, w);
    const float* l = logits + (size_t)rule.row * n;
    const int i0 = chunk_begin(n, c, chunks), i1 = chunk_begin(n, c + 1, chunks);
    const Short row = short_row<CT>(r.group_max, groups, w, bins, rule, h, sh);
    if (tid == 0) sh.n_list = 0;
    if (c == 0 && tid == 0) r.is_short = row.last < 0 ? 0 : row.all ? 2 : 1;
    if (row.last >= 0) {
        if (row.all) {
            const u64 sum = range_mass<CT>(l, i0, i1, w, bins, sh);
            if (tid == 0) atomicAdd(&r.mass[0], sum);
        }
        __syncthreads();
        range_gather<CT>(l, i0, i1, bins, 0, row.last, r.list, &r.n_list, h.mass, sh, [](int) { return true; });
        return;
    }
    range_hist<CT>(l, i0, i1, w, bins, rule.top_k > 0, h);
    for (int b = tid; b < SMP_BINS; b += CT) {
        if (h.mass[b]) atomicAdd(&r.mass[b], h.mass[b]);
        if (h.count[b]) atomicAdd(&r.count[b], h.count[b]);
    }
}

__global__ __launch_bounds__(CT) void k_smp_gather(const float* logits, int n, int bits, SmpRules rules, SmpRow* rows) {
    __shared__ Small sh;
    __shared__ u64 near[SMP_BINS];
    const int c = blockIdx.x, chunks = gridDim.x, tid = threadIdx.x;
    const SmpRule rule = rules.r[blockIdx.y];
    SmpRow& r = rows[blockIdx.y];
    const Stat s = row_stat(r, chunks);
    if (!drawn(s, rule) || r.is_short) return;
    const Weights w = weights_of(s, rule, bits);
    const Bins bins = bins_of(s, w);
    const Running<CT> run(r.mass, r.count, sh);
    const SmpCuts cuts = find_cuts<CT>(w, bins, rule, run, sh);
    if (c == 0) {  // for the last step
        run.store(r.run_mass, r.run_count);
        if (tid == 0) r.cuts = cuts;
    }
    if (tid == 0) sh.n_list = 0;
    __syncthreads();
    range_gather<CT>(logits + (size_t)rule.row * n, chunk_begin(n, c, chunks), chunk_begin(n, c + 1, chunks), bins, cuts,
                     r.list, &r.n_list, near, sh);
}

__global__ __launch_bounds__(PT) void k_smp_pick(const float* logits, int n, int bits, SmpRules rules, const SmpRow* rows,
                                                 int chunks, int32_t* tokens) {
    __shared__ Small sh;
    __shared__ union {
        PickShared p;
        SlowShared slow;
    } u;
    const SmpRule rule = rules.r[blockIdx.x];
    const SmpRow& r = rows[blockIdx.x];
    const int tid = threadIdx.x, at = rule.row;
    const u64 key = r.list[tid];
    const Stat s = row_stat(r, chunks);
    const unsigned listed = r.n_list;
    if (!drawn(s, rule)) {
        if (tid == 0) tokens[at] = token_of_undrawn(s);
        return;
    }
    const Weights w = weights_of(s, rule, bits);
    const Bins bins = bins_of(s, w);
    const int is_short = r.is_short;
    const SmpCuts cuts = is_short ? short_cuts(rule, is_short == 2 ? r.mass[0] : 0) : r.cuts;
    const u64* mass = is_short ? nullptr : r.run_mass;
    int t;
    if (listed <= 64) {
        if (tid >= 64) return;
        t = pick_wave(w, bins, rule, cuts, mass, r.run_count, key, listed);
    } else if (listed <= SMP_LIST) {
        for (int i = tid; i < (int)listed; i += PT) u.p.list[i] = i < PT ? key : r.list[i];
        __syncthreads();
        t = listed <= PT ? pick<1>(w, bins, rule, cuts, mass, r.run_count, listed, u.p, sh)
                         : pick<SMP_LIST / PT>(w, bins, rule, cuts, mass, r.run_count, listed, u.p, sh);
    } else {
        t = slow_row(logits + (size_t)at * n, n, w, bins, rule, u.slow, sh);
    }
    if (tid == 0) tokens[at] = t;
}

}  // namespace

int launch_sample_rows(const float* logits, int n_rows, int vocab, const SmpRules& rules, SmpRow* scratch, int32_t* tokens,
                       hipStream_t s) {
    const int bits = smp_bits(vocab), chunks = smp_chunks(n_rows, vocab);
    if (chunks == 0) {
        hipLaunchKernelGGL(k_smp_row, dim3(n_rows), dim3(PT), 0, s, logits, vocab, bits, rules, tokens);
    } else {
        const dim3 grid(chunks, n_rows);
        // threads that share a group: a power of two, and 512 to 1023 groups a row
        int group = 1;
        while (chunks * CT / group >= SMP_GROUPS) group *= 2;
        hipLaunchKernelGGL(k_smp_stat, grid, dim3(CT), 0, s, logits, vocab, bits, group, rules, scratch);
        // rows are in the order of their work: where the first takes the largest logit, all do
        const bool greedy = rules.r[0].temperature == 0.0f;
        if (!greedy) hipLaunchKernelGGL(k_smp_hist, grid, dim3(CT), 0, s, logits, vocab, bits, chunks * CT / group, rules, scratch);
        if (!greedy) hipLaunchKernelGGL(k_smp_gather, grid, dim3(CT), 0, s, logits, vocab, bits, rules, scratch);
        hipLaunchKernelGGL(k_smp_pick, dim3(n_rows), dim3(PT), 0, s, logits, vocab, bits, rules, (const SmpRow*)scratch, chunks,
                           tokens);
    }
    GH_HIP(hipGetLastError());
    return GH_OK;
}

}  // namespace gh
