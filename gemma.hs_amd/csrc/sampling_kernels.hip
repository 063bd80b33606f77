// gfx950 kernels of the batched sampler (temperature, top-k, top-p, min-p).
#include <hip/hip_runtime.h>

#include "sampling.h"

namespace gh {

namespace {

constexpr int NT = 1024;

typedef unsigned long long u64;

// Ascending in rank order: value descending, then index ascending.
__device__ __forceinline__ uint32_t value_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);  // -0 ranks as 0
    return (b & 0x80000000u) ? b : ~(b | 0x80000000u);
}
__device__ __forceinline__ u64 rank_key(float v, int i) { return ((u64)value_key(v) << 32) | (unsigned)i; }

// A row's weights exp((l - max) / T), as integers of `bits` fractional bits:
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

__device__ __forceinline__ u64 shfl_xor64(u64 v, int o) {
    const unsigned lo = __shfl_xor((unsigned)v, o, 64), hi = __shfl_xor((unsigned)(v >> 32), o, 64);
    return ((u64)hi << 32) | lo;
}

struct Shared {
    u64 mass[256];
    unsigned count[256];
    u64 red[NT / 64];
    u64 key, base_mass;
    unsigned base_count;
};

template <class Op>
__device__ u64 block_reduce(u64 v, Shared& sh, Op op) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = op(v, shfl_xor64(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh.red[0];
    for (int i = 1; i < NT / 64; ++i) v = op(v, sh.red[i]);
    return v;
}

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
        for (int i = tid; i < n; i += NT) {
            const u64 key = rank_key(l[i], i);
            if (shift < 56 && (key >> (shift + 8)) != (prefix >> (shift + 8))) continue;
            const int d = (int)(key >> shift) & 255;
            atomicAdd(&sh.count[d], 1u);
            const u64 m = w.fixed(l[i]);
            if (m) atomicAdd(&sh.mass[d], m);
        }
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

__global__ __launch_bounds__(NT) void k_sample_row(const float* logits, int n, double one, SmpRules rules, int32_t* tokens) {
    __shared__ Shared sh;
    const gh_sampling rule = rules.r[blockIdx.x];
    const float* l = logits + (size_t)blockIdx.x * n;
    const int tid = threadIdx.x;
    // the first in rank order; a NaN is known by its own bit
    u64 first = ~0ull, nan = 0;
    for (int i = tid; i < n; i += NT) {
        if (l[i] != l[i]) nan = 1;
        else if (l[i] > -INFINITY) first = min(first, rank_key(l[i], i));
    }
    first = block_reduce(first, sh, [](u64 a, u64 b) { return a < b ? a : b; });
    nan = block_reduce(nan, sh, [](u64 a, u64 b) { return a | b; });
    if (nan || first == ~0ull || rule.temperature == 0.0f) {
        if (tid == 0) tokens[blockIdx.x] = nan || first == ~0ull ? -1 : (int)(unsigned)first;
        return;
    }
    const Weights w{l[(unsigned)first], 1.0 / (double)rule.temperature, one};
    u64 total = 0, at_least = 0;
    for (int i = tid; i < n; i += NT) {
        const u64 m = w.fixed(l[i]);
        total += m;
        if (w.real(l[i]) >= (double)rule.min_p) at_least += m;
    }
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
    if (tid == 0) tokens[blockIdx.x] = (int)(unsigned)sh.key;
}

}  // namespace

int launch_sample_rows(const float* logits, int n_rows, int vocab, const SmpRules& rules, int32_t* tokens, hipStream_t s) {
    hipLaunchKernelGGL(k_sample_row, dim3(n_rows), dim3(NT), 0, s, logits, vocab, ldexp(1.0, smp_bits(vocab)), rules, tokens);
    GH_HIP(hipGetLastError());
    return GH_OK;
}

}  // namespace gh
