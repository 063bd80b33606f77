// gfx950 kernels of the 8-bit KV cache: quantising append, truncation,
// read-back, and the attention that reads the codes on the int8 matrix cores.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "kv8.h"

namespace gh {

namespace {

constexpr int NT = 256;  // threads per workgroup (4 wave64)

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
constexpr uint32_t INF_BITS = 0x7f800000u;

// Max over the workgroup (one barrier before, one after; `slot`: 16 words of LDS).
template <int THREADS>
__device__ __forceinline__ uint32_t block_max_u32(uint32_t v, uint32_t* slot) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    v = slot[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) v = max(v, slot[w]);
    return v;
}

// ------------------------------------------------------------------
// quantisation of one block (64 tokens of one kv head), one workgroup
// ------------------------------------------------------------------
// Scale of values whose largest magnitude has these bits; NaN where one of
// them is not finite (an int8 cannot hold it, and a wrong number would not
// show).  2^-100 keeps the scale, and half of it, a normal number.
__device__ __forceinline__ float scale_of(uint32_t a) {
    return a >= INF_BITS ? __uint_as_float(0x7fc00000u) : fmaxf(__uint_as_float(a) / 127.0f, 0x1p-100f);
}

// x / s rounded half to even, exactly.  c = rint(x * inv) is off by one at
// most, and only near the middle between two codes; x - c s fits into 24
// bits there (a multiple of the smaller ulp, no larger than s / 2 and a bit),
// so one fma gives it without rounding and its comparison with s / 2 decides.
// A NaN scale gives 0.
__device__ __forceinline__ int code_of(float x, float s, float inv) {
    const float c = rintf(x * inv), r = fmaf(-c, s, x), h = 0.5f * s;
    int k = (int)c;
    if (fabsf(r) > h || (fabsf(r) == h && (k & 1))) k += r > 0.0f ? 1 : -1;
    return s == s ? k : 0;
}

// A block as one workgroup takes it, 16 values a thread.  K: 4 dims of rows
// row, row + 16, ..., whole rows a load instruction; V: 16 rows of one dim,
// whose codes are 16 consecutive bytes (the layout in kv8.h).  The f32 rows
// pass by the caches, which have no use for them: prompts of 16 sequences
// appended and read back in 120 us, 141 without.
template <int HD, bool V>
struct Item {
    static constexpr int N = 4 * HD;  // the workgroup's threads
    int row, col;  // first row, first dim
    __device__ __forceinline__ explicit Item(int e) {
        row = V ? e / HD * 4 : e / (HD / 4);
        col = V ? e % HD : e % (HD / 4) * 4;
    }
    // byte offset of a value's code
    __device__ __forceinline__ static int place(int r, int d) {
        if (V) return ((d / 16) * 64 + (r / 4 % 4) * 16 + d % 16) * 16 + r / 16 * 4 + r % 4;
        constexpr int KD = HD < 64 ? 1 : HD / 64;
        return ((r / 16 * KD + d / 64) * 64 + (d / 16 % 4) * 16 + r % 16) * 16 + d % 16;
    }
    // row of value j
    __device__ __forceinline__ int row_of(int j) const { return row + 16 * (j / 4) + (V ? j % 4 : 0); }
};

// The item's values of rows [lo, hi) from src (row 0, `ld` floats a row: a
// block is below 2^31 bytes); the others as they are.  A row out of reach is
// replaced by one within for the load, so that no load waits for a branch.
template <int HD, bool V>
__device__ __forceinline__ void load_item(const Item<HD, V>& it, const float* src, uint32_t ld, int lo, int hi, float (&x)[16]) {
    const char* base = (const char*)(src + (ptrdiff_t)lo * (ptrdiff_t)ld);
    auto at = [&](int j) { return base + 4 * ((uint32_t)(min(max(it.row_of(j), lo), hi - 1) - lo) * ld + it.col); };
    auto in = [&](int j) { return it.row_of(j) >= lo && it.row_of(j) < hi; };
    if (V) {
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = __builtin_nontemporal_load((const float*)at(j));
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = in(j) ? v[j] : x[j];
    } else {
        f32x4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __builtin_nontemporal_load((const f32x4*)at(4 * j));
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = in(j) ? v[j / 4][j % 4] : x[j];
    }
}

// The item's values of rows [lo, hi) to dst (row 0, `ld` floats a row).
template <int HD, bool V>
__device__ __forceinline__ void store_item(const Item<HD, V>& it, float* dst, size_t ld, int lo, int hi, const float (&x)[16]) {
    auto at = [&](int j) { return dst + (ptrdiff_t)it.row_of(j) * (ptrdiff_t)ld + it.col; };
#pragma unroll
    for (int j = 0; j < 16; j += V ? 1 : 4) {
        const int r = it.row_of(j);
        if (r < lo || r >= hi) continue;
        if (V) __builtin_nontemporal_store(x[j], at(j));
        else __builtin_nontemporal_store(f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]}, (f32x4*)at(j));
    }
}

// The 16 codes as bytes.  x * inv + 1.5 2^23 has the code in its low byte, and
// the only error before its rounding is inv's, below 127 2^-24: unless a
// quotient lies within 2^-16 of the middle between two codes (a wave in
// thirty), that is the answer.
__device__ __forceinline__ i32x4 codes_of(const float (&x)[16], float s) {
    constexpr float MAGIC = 0x1.8p23f;
    const float inv = 1.0f / s;
    uint32_t v[16];
    float off = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const float t = fmaf(x[j], inv, MAGIC);
        off = fmaxf(off, fabsf(fmaf(x[j], inv, MAGIC - t)));
        v[j] = __float_as_uint(t);
    }
    if (__any(off > 0.5f - 0x1p-16f)) {
#pragma unroll 1
        for (int j = 0; j < 16; ++j) v[j] = (uint32_t)code_of(x[j], s, inv);
    }
    i32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t lo = __builtin_amdgcn_perm(v[4 * j + 1], v[4 * j], 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(v[4 * j + 3], v[4 * j + 2], 0x04000c0cu);
        w[j] = (int)(lo | hi);
    }
    return w;
}

template <int HD, bool V>
__device__ __forceinline__ void store_codes(const Item<HD, V>& it, int8_t* block, float s, const float (&x)[16]) {
    const i32x4 w = codes_of(x, s);
    if (V) *(i32x4*)(block + Item<HD, V>::place(it.row, it.col)) = w;
#pragma unroll
    for (int j = 0; !V && j < 4; ++j) *(int*)(block + Item<HD, V>::place(it.row_of(4 * j), it.col)) = w[j];
}

// f32 values of the codes: one product each, rounded once
template <int HD, bool V>
__device__ __forceinline__ void read_item(const Item<HD, V>& it, const int8_t* block, float s, float (&x)[16]) {
    union {
        int8_t b[16];
        int i[4];
        i32x4 w;
    } u;
    if (V) u.w = *(const i32x4*)(block + Item<HD, V>::place(it.row, it.col));
#pragma unroll
    for (int j = 0; !V && j < 4; ++j)
        u.i[j] = *(const int*)(block + Item<HD, V>::place(it.row_of(4 * j), it.col));
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = (float)u.b[j] * s;
}

__device__ __forceinline__ uint32_t amax(const float (&x)[16]) {
    uint32_t a = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) a = max(a, abs_bits(x[j]));
    return a;
}

// Rows [r0, r1) of a block come from src (its row 0), the first r0 are there
// already: codes, scale, and with `keep` the f32 rows of the new ones.
template <int HD, bool V>
__device__ __forceinline__ void append_block(int8_t* block, float* scale, float* tail, const float* src, size_t ld, int r0,
                                             int r1, bool keep, uint32_t* slot) {
    constexpr int N = Item<HD, V>::N;
    const int tid = threadIdx.x;
    float s = 0.0f;
    if (r0 > 0) {
        // A few rows behind others: if they do not raise the scale, theirs
        // are the only codes to write.
        const float old = *scale;
        uint32_t a = 0;
        const int e1 = (r1 - r0) * HD;
        for (int e = tid; e < e1; e += N) a = max(a, abs_bits(src[(ptrdiff_t)(r0 + e / HD) * (ptrdiff_t)ld + e % HD]));
        s = scale_of(block_max_u32<N>(a, slot));  // its barriers: every thread has read the old scale
        if (old != old || s != s) s = __uint_as_float(0x7fc00000u);
        else s = fmaxf(s, old);
        if (tid == 0) *scale = s;
        const bool same = !(s > old);
        if (same || keep) {
            const float inv = 1.0f / s;
            for (int e = tid; e < e1; e += N) {
                const int r = r0 + e / HD, d = e % HD;
                const float x = src[(ptrdiff_t)r * (ptrdiff_t)ld + d];
                if (same) block[Item<HD, V>::place(r, d)] = (int8_t)code_of(x, s, inv);
                if (keep) tail[r * HD + d] = x;
            }
        }
        if (same) return;
    }
    const Item<HD, V> it(tid);
    float x[16] = {};
    load_item<HD, V>(it, src, ld, r0, r1, x);
    if (r0 > 0) {
        load_item<HD, V>(it, tail, HD, 0, r0, x);
    } else {
        s = scale_of(block_max_u32<N>(amax(x), slot));
        if (tid == 0) *scale = s;
        if (keep) store_item<HD, V>(it, tail, HD, 0, r1, x);
    }
    store_codes<HD, V>(it, block, s, x);
}

// One workgroup per block that the new tokens touch, kv head and K or V.
// Reads 4 bytes an element and writes 1: bound by memory.  Prompts of up to
// 1920 tokens for 16 sequences, 4 kv heads of 256 dims: 54 us, 5.1 TB/s of
// both (a large copy reaches 5.1).  One token is the latency of its loads and
// barriers, 3.3 us.
template <int HD>
__global__ __launch_bounds__(4 * HD, 8) void k_kv8_append(Kv8Dev c, Kv8Batch b, const float* k, const float* v) {
    __shared__ uint32_t slot[16];
    const int i = blockIdx.z, h = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    const int pos = b.pos[i], cnt = b.cnt[i], end = pos + cnt;
    const int first = pos / KV8_BLOCK, blk = first + blockIdx.x;
    if (cnt == 0 || blk * KV8_BLOCK >= end) return;
    const int r0 = max(pos - blk * KV8_BLOCK, 0), r1 = min(end - blk * KV8_BLOCK, KV8_BLOCK);
    const size_t ld = (size_t)c.nkv * HD, head = (size_t)b.seq[i] * c.nkv + h, at = head * c.nb + blk;
    // row 0 of the block (in front of the input where the block holds tokens already)
    const float* in = is_v ? v : k;
    const float* src = in + ((ptrdiff_t)b.off[i] + (blk * KV8_BLOCK - pos)) * (ptrdiff_t)ld + h * HD;
    float* tail = (is_v ? c.vt : c.kt) + head * KV8_BLOCK * HD;
    // The f32 rows of the last block, if it is not full.  Where the first
    // block needs the old ones, its workgroup puts the new ones there, after
    // it has read them.
    const bool shared_tail = pos % KV8_BLOCK != 0 && (end - 1) / KV8_BLOCK != first;
    const bool keep = r1 < KV8_BLOCK && !(shared_tail && blk != first);
    if (is_v)
        append_block<HD, true>(c.vc + at * KV8_BLOCK * HD, c.vs + at, tail, src, ld, r0, r1, keep, slot);
    else
        append_block<HD, false>(c.kc + at * KV8_BLOCK * kv8_k_row(HD), c.ks + at, tail, src, ld, r0, r1, keep, slot);
    const int left = end % KV8_BLOCK;
    if (shared_tail && blk == first && left) {
        __syncthreads();
        const float* from = in + ((size_t)b.off[i] + cnt - left) * ld + h * HD;
        for (int e = threadIdx.x; e < left * (HD / 4); e += 4 * HD)
            ((f32x4*)tail)[e] = *(const f32x4*)(from + (size_t)(e / (HD / 4)) * ld + e % (HD / 4) * 4);
    }
}

// A block that keeps its first r1 rows.  same: it was the last one already,
// its f32 rows are there and are quantised anew; else its values become them.
template <int HD, bool V>
__device__ __forceinline__ void truncate_block(int8_t* block, float* scale, float* tail, int r1, bool same, uint32_t* slot) {
    const Item<HD, V> it(threadIdx.x);
    float x[16] = {};
    if (same) {
        load_item<HD, V>(it, tail, HD, 0, r1, x);
        const float s = scale_of(block_max_u32<Item<HD, V>::N>(amax(x), slot));
        if (threadIdx.x == 0) *scale = s;
        store_codes<HD, V>(it, block, s, x);
    } else {
        read_item<HD, V>(it, block, *scale, x);
        store_item<HD, V>(it, tail, HD, 0, r1, x);
    }
}

// One workgroup per kv head and K or V: latency, 3.9 us for one sequence, 6.6
// for 31 of 4 kv heads.
template <int HD>
__global__ __launch_bounds__(4 * HD, 8) void k_kv8_truncate(Kv8Dev c, Kv8Batch b) {
    __shared__ uint32_t slot[16];
    const int i = blockIdx.z, h = blockIdx.y >> 1;
    const int blk = b.cnt[i] / KV8_BLOCK, r1 = b.cnt[i] % KV8_BLOCK;
    const bool same = blk == b.pos[i] / KV8_BLOCK;
    const size_t head = (size_t)b.seq[i] * c.nkv + h, at = head * c.nb + blk;
    if (blockIdx.y & 1)
        truncate_block<HD, true>(c.vc + at * KV8_BLOCK * HD, c.vs + at, c.vt + head * KV8_BLOCK * HD, r1, same, slot);
    else
        truncate_block<HD, false>(c.kc + at * KV8_BLOCK * kv8_k_row(HD), c.ks + at, c.kt + head * KV8_BLOCK * HD, r1, same,
                                  slot);
}

// As k_kv8_append, 1 byte read and 4 written: 41 us for its prompts, 6.6 TB/s.
template <int HD>
__global__ __launch_bounds__(4 * HD, 8) void k_kv8_read(Kv8Dev c, Kv8Batch b, float* k, float* v) {
    const int i = blockIdx.z, h = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    float* out = is_v ? v : k;
    const int pos = b.pos[i], cnt = b.cnt[i], end = pos + cnt;
    const int blk = pos / KV8_BLOCK + blockIdx.x;
    if (!out || cnt == 0 || blk * KV8_BLOCK >= end) return;
    const int r0 = max(pos - blk * KV8_BLOCK, 0), r1 = min(end - blk * KV8_BLOCK, KV8_BLOCK);
    const size_t ld = (size_t)c.nkv * HD, at = ((size_t)b.seq[i] * c.nkv + h) * c.nb + blk;
    float* dst = out + ((ptrdiff_t)b.off[i] + (blk * KV8_BLOCK - pos)) * (ptrdiff_t)ld + h * HD;  // row 0 of the block
    float x[16];
    if (is_v) {
        const Item<HD, true> it(threadIdx.x);
        read_item<HD, true>(it, c.vc + at * KV8_BLOCK * HD, c.vs[at], x);
        store_item<HD, true>(it, dst, ld, r0, r1, x);
    } else {
        const Item<HD, false> it(threadIdx.x);
        read_item<HD, false>(it, c.kc + at * KV8_BLOCK * kv8_k_row(HD), c.ks[at], x);
        store_item<HD, false>(it, dst, ld, r0, r1, x);
    }
}

// ------------------------------------------------------------------
// attention
// ------------------------------------------------------------------
// Products of the codes run on the int8 matrix cores, which sum them exactly.
// The other operand, a row of q or of probabilities, is an integer of 23 bits
// and sign, relative to the row's (or block's) largest magnitude, in three
// signed digits to the base 256: with L = 127 (65536 + 256 + 1) the largest
// such integer, x = a / L * (65536 d2 + 256 d1 + d0), off by at most a / 2 L
// (2^-24 a: what rounding a to f32 costs).  Three products give the integer
// dot product; no code is ever converted.
constexpr float DIGIT_MAX = 8355711.0f;
// Digits of v, |v| <= DIGIT_MAX, as the three low bytes, 128 too large: adding
// 128 (65536 + 256 + 1) makes every digit an unsigned byte.
__device__ __forceinline__ uint32_t digits_of(float v) { return (uint32_t)((int)rintf(v) + 0x808080); }
// The same for m p with 0 <= p <= 1, m <= DIGIT_MAX, the two low digits 128 too
// large: an f32 between 2^23 and 2^24 has its integer in its low bits, and the sum
// below stays in front of 2^24.
__device__ __forceinline__ uint32_t digits_of_share(float p, float m) { return __float_as_uint(fmaf(p, m, 0x1p23f + 0x8080)); }
constexpr uint32_t DIGIT_BIAS = 0x80808080u;  // what an exclusive or takes off four digits that are 128 too large

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
constexpr int DPP_ROW_ROR4 = 0x124, DPP_ROW_ROR8 = 0x128;

__device__ __forceinline__ i32x4 mfma(i32x4 a, i32x4 b, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// a b as a number of its own: not part of a fused addition
__device__ __forceinline__ float rounded(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

// byte n of four words
__device__ __forceinline__ uint32_t byte_of(const uint32_t* d, int n) {
    const uint32_t lo = __builtin_amdgcn_perm(d[1], d[0], n == 0 ? 0x0c0c0400u : n == 1 ? 0x0c0c0501u : 0x0c0c0602u);
    const uint32_t hi = __builtin_amdgcn_perm(d[3], d[2], n == 0 ? 0x04000c0cu : n == 1 ? 0x05010c0cu : 0x06020c0cu);
    return lo | hi;
}

// The query rows of a workgroup: ROWS (token, head) pairs of one kv head, and
// the chunk of key blocks that they look at.
template <int ROWS>
struct Tile {
    const Kv8Batch& b;
    const Att8& a;
    int i, h, chunk;  // entry, kv head, chunk
    int row0, rows;   // first row, and how many there are
    int first;        // position of the entry's first query token
    int p0, p1;       // positions of the tile's first and last row
    int blk0, blk1;   // key blocks
    __device__ __forceinline__ Tile(const Kv8Batch& b, const Att8& a, int i, int h, int chunk, int tile)
        : b(b), a(a), i(i), h(h), chunk(chunk), row0(tile * ROWS) {
        const int n_q = b.cnt[i];
        rows = min(n_q * a.group - row0, ROWS);
        first = b.pos[i] - n_q;
        p0 = first + token_of(0);
        p1 = first + token_of(rows - 1);
        // the blocks that they see, in chunks of one size: as many as a.chunk makes, evenly
        const int begin = a.window ? max(p0 - a.window + 1, 0) / KV8_BLOCK : 0, end = p1 < 0 ? 0 : p1 / KV8_BLOCK + 1;
        const unsigned blocks = max(end - begin, 0), parts = (blocks + a.chunk - 1) / (unsigned)a.chunk;
        const int size = a.ns > 1 && parts ? (int)((blocks + parts - 1) / parts) : (int)blocks;
        blk0 = begin + chunk * size;
        blk1 = min(blk0 + size, end);
    }
    // query token of row r, and the row's place in q and out
    __device__ __forceinline__ int token_of(int r) const {
        return (int)__umulhi((unsigned)(row0 + r), a.group_inv) + (a.group == 1 ? row0 + r : 0);
    }
    __device__ __forceinline__ size_t slot_of(int r) const {
        const int t = token_of(r);
        return ((size_t)b.off[i] + t) * a.heads + (h * a.group + row0 + r - t * a.group);
    }
    // and among the chunk states
    __device__ __forceinline__ size_t part_of(int r) const {
        return slot_of(r) + ((ptrdiff_t)b.part[i] - b.off[i]) * a.heads;
    }
    // a chunk with nothing to see
    template <int HD>
    __device__ __forceinline__ void put_nothing(int tid, int threads) const {
        if (a.ns > 1) {
            if (tid < rows) {
                a.part[part_of(tid) * a.ns + chunk] = -INFINITY;
                a.part[(a.rows + part_of(tid)) * a.ns + chunk] = 0.0f;
            }
        } else {
            for (int e = tid; e < rows * HD; e += threads) a.out[slot_of(e / HD) * HD + e % HD] = 0.0f;
        }
    }
    // dims 4 q4 .. of row r: v, with the maximum M and the sum L that go with it
    template <int HD>
    __device__ __forceinline__ void put(int r, int q4, f32x4 v, float M, float L) const {
        if (a.ns > 1) {
            const size_t at = part_of(r) * a.ns + chunk;
            if (q4 == 0) {
                a.part[at] = M;
                a.part[a.rows * a.ns + at] = L;
            }
            ((f32x4*)(a.part + 2 * a.rows * a.ns + at * HD))[q4] = v;
        } else {
            ((f32x4*)(a.out + slot_of(r) * HD))[q4] = v * (M == -INFINITY && L == 0.0f ? 0.0f : 1.0f / L);
        }
    }
    // not every row sees all of the block
    __device__ __forceinline__ bool masked(int blk) const {
        return blk * KV8_BLOCK + KV8_BLOCK - 1 > p0 || (a.window && blk * KV8_BLOCK < p1 - a.window + 1);
    }
};

// Digits of the tile's query rows into the columns of Cols (a wave a row, a
// lane 4 dims), and the rows' largest magnitudes.  Ends with a barrier.
template <int HD, class Cols, int N>
__device__ __forceinline__ void put_queries(const Tile<Cols::ROWS>& tile, i32x4 (&qs)[N][kv8_k_row(HD) / 64][64],
                                            uint32_t (&qmax)[Cols::ROWS], int lane, int wave) {
    constexpr int KR = kv8_k_row(HD), ROWS = Cols::ROWS, WAVES = Cols::WAVES, RW = (ROWS + WAVES - 1) / WAVES;
    f32x4 x[RW];
#pragma unroll
    for (int e = 0; e < RW; ++e) {
        const int r = wave + e * WAVES;
        x[e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (r < tile.rows && 4 * lane < HD) x[e] = ((const f32x4*)(tile.a.q + tile.slot_of(r) * HD))[lane];
    }
#pragma unroll
    for (int e = 0; e < RW; ++e) {
        const int r = wave + e * WAVES;
        if (ROWS % WAVES && r >= ROWS) break;
        uint32_t m = max(max(abs_bits(x[e].x), abs_bits(x[e].y)), max(abs_bits(x[e].z), abs_bits(x[e].w)));
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
        // a row that is nearly zero: its digits vanish
        const float inv = DIGIT_MAX / fmaxf(__uint_as_float(m), 0x1p-100f);
        uint32_t dg[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) dg[d] = digits_of(fminf(fmaxf(x[e][d] * inv, -DIGIT_MAX), DIGIT_MAX));
        if (4 * lane < KR) {
#pragma unroll
            for (int n = 0; n < Cols::PLACES; ++n)
                ((uint32_t*)&qs[Cols::operand(n)][lane >> 4][(lane >> 2 & 3) * 16 + Cols::place(r, n)])[lane & 3] =
                    n < 3 ? byte_of(dg, n) ^ DIGIT_BIAS : 0u;
        }
        if (lane == 0) qmax[r] = m;
    }
    __syncthreads();
}

// What turns a row's integer products into scores q . k / sqrt(HD) in units of
// ln 2, but for the scale of K; NaN for a row that is not finite.
template <int HD>
__device__ __forceinline__ float query_scale(uint32_t m) {
    constexpr float ROOT = HD == 32 ? 5.65685424949238f : HD == 64 ? 8.0f : HD == 128 ? 11.3137084989848f : 16.0f;
    return m >= INF_BITS ? __uint_as_float(0x7fc00000u)
                         : fmaxf(__uint_as_float(m), 0x1p-100f) * (1.44269504088896340736f / DIGIT_MAX / ROOT);
}

// The 16 columns of a product where a kv head has few query rows (decoding): 4
// rows with their three digits side by side, column 4 n + r digit n of row r
// and the last four zero.  A third of the products, and of the conversions of
// their results, that a product for each digit would take.
struct Narrow {
    static constexpr int ROWS = 4, WAVES = 8, PLACES = 4;
    int row, digit;
    uint32_t lo, hi, bias;  // byte selectors of the lane's digit, and what its bytes are too large
    float weight;
    // each code is read once a call
    __device__ __forceinline__ static i32x4 load(const i32x4* p) { return __builtin_nontemporal_load(p); }
    __device__ __forceinline__ explicit Narrow(int col) : row(col & 3), digit(col >> 2) {
        lo = digit == 3 ? 0x0c0c0c0cu : 0x0c0c0400u + 0x0101u * digit;
        hi = digit == 3 ? 0x0c0c0c0cu : 0x04000c0cu + 0x01010000u * digit;
        bias = digit < 2 ? DIGIT_BIAS : 0u;
        weight = digit == 0 ? 1.0f : digit == 1 ? 256.0f : 65536.0f;
    }
    // the lane's digit of four probabilities
    __device__ __forceinline__ int share(const uint32_t* d) const {
        return (int)((__builtin_amdgcn_perm(d[1], d[0], lo) | __builtin_amdgcn_perm(d[3], d[2], hi)) ^ bias);
    }
    // column of digit n of a query row
    __device__ __forceinline__ static int place(int r, int n) { return 4 * n + r; }
    __device__ __forceinline__ static int operand(int) { return 0; }
    // The row's value from its digits' ones.  Its lanes have to get the same sum to the last bit, since each
    // takes its own digit of the probability that comes of it: additions of
    // the same values in either order, none fused with the product before.
    __device__ __forceinline__ float join(float v) const {
#pragma clang fp contract(off)
        v = v + dpp<DPP_ROW_ROR8>(v);
        return v + dpp<DPP_ROW_ROR4>(v);
    }
};

// One workgroup: up to four query rows of one kv head x one chunk of key
// blocks, the blocks dealt to its waves; each wave keeps its own running
// maximum, sum and output, joined through LDS at the end.
//   S^T = K Q^T   operand A: codes of 16 tokens, B: digits of the query rows;
//                 lane (g, col) gets tokens 16 t + 4 g + i of its row
//   O^T = V^T P^T operand A: codes of 16 dims, B: digits of the lane's own
//                 16 probabilities (the layout of V has their order)
// The codes of the next block are on their way while the present one is
// worked on, as far as the registers reach.
// Bound by memory where there are enough sequences: 64 of some 4000 tokens, 4
// kv heads of 256 dims 91 us, 6.1 TB/s (a plain read reaches 6.8 to 7.2);
// their codes pass by the caches (116 us a call without, 106 so).  Else by the
// chain from a load to the output: 7 us for 512 tokens of one kv head, 13 for
// 32768 of four in 64 chunks each, and 4 to join these.
template <int HD>
__global__ __launch_bounds__(64 * Narrow::WAVES, 2) void k_kv8_attention(Kv8Dev c, Kv8Batch b, Att8 a) {
    constexpr int KR = kv8_k_row(HD), KD = KR / 64, VD = HD / 16, ROWS = Narrow::ROWS, WAVES = Narrow::WAVES;
    constexpr bool LATE_K = HD == 256;  // K and V early do not fit its registers
    __shared__ float st_m[WAVES][ROWS], st_l[WAVES][ROWS];
    __shared__ uint32_t qmax[ROWS];
    __shared__ i32x4 qs[1][KD][64];
    __shared__ __align__(16) float ob[WAVES][ROWS][HD + 4];
    // grid: chunks, kv heads, entries.  Neighbours in the grid go to different
    // XCDs; each entry and head begins with another chunk, so that those of
    // one chunk do not all meet on one (31 sequences of 1000 tokens beside one
    // of 32768, 8 kv heads: 142 us, turned 51).
    const int i = blockIdx.z, h = blockIdx.y;
    const unsigned turned = blockIdx.x + (blockIdx.y + blockIdx.z) % (unsigned)a.ns;
    const Tile<ROWS> tile(b, a, i, h, turned < (unsigned)a.ns ? turned : turned - a.ns, 0);
    const int rows = tile.rows, blk1 = tile.blk1;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    const Narrow col(lane & 15);
    if (tile.blk0 >= blk1) return tile.put_nothing<HD>(tid, 64 * WAVES);
    const size_t head = ((size_t)b.seq[i] * c.nkv + h) * c.nb;
    i32x4 kk[4][KD], vv[VD];
    float ks, vs;
    auto load_k = [&](int blk) {
        const i32x4* p = (const i32x4*)(c.kc + (head + blk) * KV8_BLOCK * KR) + lane;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int d = 0; d < KD; ++d) kk[t][d] = Narrow::load(p + (t * KD + d) * 64);
        ks = c.ks[head + blk];
    };
    auto load_v = [&](int blk) {
        const i32x4* p = (const i32x4*)(c.vc + (head + blk) * KV8_BLOCK * HD) + lane;
#pragma unroll
        for (int d = 0; d < VD; ++d) vv[d] = Narrow::load(p + d * 64);
        vs = c.vs[head + blk];
    };
    int blk = tile.blk0 + wave;
    if (blk < blk1) {
        load_k(blk);
        load_v(blk);
    }
    put_queries<HD, Narrow>(tile, qs, qmax, lane, wave);
    const float qscale = query_scale<HD>(qmax[col.row]) * col.weight;
    const int pos = col.row < rows ? tile.first + tile.token_of(col.row) : -1;
    const int from = a.window ? pos - a.window + 1 : 0;
    float m_run = -INFINITY, l_run = 0.0f;
    f32x4 o[VD];
#pragma unroll
    for (int d = 0; d < VD; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (; blk < blk1; blk += WAVES) {
        int at = lane;
        asm volatile("" : "+v"(at));  // q's digits are read again for each block: no registers to keep them in
        const float f = qscale * ks;
        float s[16], mb = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            i32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int d = 0; d < KD; ++d) acc = mfma(kk[t][d], qs[0][d][at], acc);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[4 * t + j] = col.join(rounded((float)acc[j], f));
        }
        if (!LATE_K && blk + WAVES < blk1) load_k(blk + WAVES);
        if (tile.masked(blk)) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int p = blk * KV8_BLOCK + 16 * (j / 4) + 4 * g + j % 4;
                s[j] = p <= pos && p >= from ? s[j] : -INFINITY;
            }
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) mb = fmaxf(mb, s[j]);
        mb = fmaxf(mb, __shfl_xor(mb, 16, 64));
        mb = fmaxf(mb, __shfl_xor(mb, 32, 64));
        // Probabilities relative to the block's own maximum.  A row that sees
        // nothing of the block has -inf for all its scores, and none of them
        // may take part whatever the block's scales are; one whose scores are
        // all NaN has the same maximum, and its sum becomes NaN.
        const float top = mb == -INFINITY ? 0.0f : mb;
        float lb = 0.0f;
        uint32_t pd[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float e = exp2_fast(s[j] - top);
            lb += e;
            pd[j] = digits_of_share(e, DIGIT_MAX);
        }
        const float m_new = fmaxf(m_run, mb);
        const float alpha = m_run == m_new ? 1.0f : exp2_fast(m_run - m_new);
        const float beta = mb == -INFINITY ? 0.0f : exp2_fast(mb - m_new);
        m_run = m_new;
        l_run = l_run * alpha + (mb == -INFINITY ? lb : lb * beta);
        const float w = mb == -INFINITY ? 0.0f : beta * vs * (1.0f / DIGIT_MAX) * col.weight;
        i32x4 pb;
#pragma unroll
        for (int t = 0; t < 4; ++t) pb[t] = col.share(pd + 4 * t);
        __builtin_amdgcn_sched_barrier(0);  // scores and probabilities leave their registers here
        if (LATE_K && blk + WAVES < blk1) load_k(blk + WAVES);
        if (__any(alpha != 1.0f)) {
#pragma unroll
            for (int d = 0; d < VD; ++d) o[d] *= alpha;
        }
#pragma unroll
        for (int d = 0; d < VD; ++d) {
            const i32x4 acc = mfma(vv[d], pb, i32x4{0, 0, 0, 0});
#pragma unroll
            for (int j = 0; j < 4; ++j) o[d][j] = fmaf((float)acc[j], w, o[d][j]);
        }
        if (blk + WAVES < blk1) load_v(blk + WAVES);
    }
    // join the waves
    l_run += __shfl_xor(l_run, 16, 64);
    l_run += __shfl_xor(l_run, 32, 64);
    if (g == 0) {
        st_m[wave][col.row] = m_run;
        st_l[wave][col.row] = l_run;
    }
    // the row's four lanes add their digits' parts; each writes a quarter (all of it where there are fewer)
    constexpr int STEP = VD < 4 ? 1 : 4;
#pragma unroll
    for (int d = 0; d < VD; d += STEP) {
        f32x4 v[STEP];
#pragma unroll
        for (int e = 0; e < STEP; ++e)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[e][j] = col.join(o[d + e][j]);
        f32x4 mine = v[0];
        if constexpr (STEP == 4) {
            const f32x4 x = col.digit & 1 ? v[1] : v[0], y = col.digit & 1 ? v[3] : v[2];
            mine = col.digit & 2 ? y : x;
        }
        *(f32x4*)&ob[wave][col.row][16 * (d + (STEP == 4 ? col.digit : 0)) + 4 * g] = mine;
    }
    __syncthreads();
    const int jr = tid / (HD / 4), q4 = tid % (HD / 4);  // row and dims that this thread joins
    if (jr >= rows) return;
    float M = -INFINITY, L = 0.0f;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) M = fmaxf(M, st_m[w][jr]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const float x = st_m[w][jr] == -INFINITY ? 0.0f : exp2_fast(st_m[w][jr] - M);
        L += st_l[w][jr] * x;
        v += *(const f32x4*)&ob[w][jr][4 * q4] * x;
    }
    tile.put<HD>(jr, q4, v, M, L);
}

// A scale that is the same for a wave, by a scalar load: a vector load would
// come back behind the codes that are on their way.
__device__ __forceinline__ float scalar_load(const float* p) {
    return *(const __attribute__((address_space(4))) float*)(uintptr_t)p;
}

// The 16 columns where a kv head has more: a query row each, a product for
// each digit.
struct Wide {
    static constexpr int ROWS = 16, WAVES = 4, PLACES = 3;
    __device__ __forceinline__ static int place(int r, int) { return r; }
    __device__ __forceinline__ static int operand(int n) { return n; }
    // the digits' products together; each is below 2^24 (256 dims, or tokens)
    __device__ __forceinline__ static float sum(int d0, int d1, int d2) {
        return fmaf((float)d2, 65536.0f, (float)(d1 * 256 + d0));
    }
};

// One workgroup: up to 16 query rows of one kv head x one chunk of key blocks,
// four blocks a step.  A wave takes one of them for the scores, and a quarter
// of the dims for all four of them: the probabilities' digits pass through
// LDS.  So the integer sums of four blocks become floats once, no wave holds
// more than a quarter of the output, and nothing is joined at the end.
// The probabilities are relative to the step's largest, and carry the block's
// share of the largest scale of V that the row sees.
// Bound by the conversions around the products and by one phase waiting for
// the other, two workgroups a CU (256 dims; three and four for 128 and 64):
// the matrix cores are busy for a third of the time, L2 gives 12 TB/s of the
// 33 that it could.  A prompt of 1907 tokens in a window of 1024, 8 heads of
// 256 dims over 4: 42 us, 4096 tokens of 32 heads of 128 over 8: 310 (445
// TFLOP/s of the formula's products; a large bf16 product reaches 1234).  By
// four waves with blocks and outputs of their own, joined at the end: 45 and
// 360, and drafts for 16 sequences of 2011 tokens 14 us (here 12.5).
// ONCE: one tile a kv head, each code is read once a call.
template <int HD, bool ONCE>
__global__ __launch_bounds__(64 * Wide::WAVES, HD == 256 ? 2 : HD == 128 ? 3 : 4) void k_kv8_attention_wide(Kv8Dev c, Kv8Batch b, Att8 a) {
    constexpr int KR = kv8_k_row(HD), KD = KR / 64, VD = HD / 16, ROWS = Wide::ROWS, WAVES = Wide::WAVES;
    constexpr int DT = VD < WAVES ? 1 : VD / WAVES;  // 16-dim tiles a wave
    __shared__ float st_m[WAVES][ROWS], st_l[WAVES][ROWS];
    __shared__ uint32_t qmax[ROWS];
    __shared__ i32x4 qs[3][KD][64], ps[WAVES][3][64];
    // grid: kv heads, then the chunks (turned as above), then the tiles, the longest (last) first; entries
    const int i = blockIdx.z;
    const unsigned by_head = blockIdx.x / (unsigned)c.nkv, by_chunk = a.ns > 1 ? by_head / (unsigned)a.ns : by_head;
    const int h = blockIdx.x - by_head * c.nkv, t0 = a.tiles - 1 - by_chunk;
    if (t0 * ROWS >= b.cnt[i] * a.group) return;
    unsigned chunk = by_head - by_chunk * a.ns;
    if (a.ns > 1) chunk = (chunk + blockIdx.z) % (unsigned)a.ns;
    const Tile<ROWS> tile(b, a, i, h, chunk, t0);
    const int blk1 = tile.blk1;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, row = lane & 15;
    if (tile.blk0 >= blk1) return tile.put_nothing<HD>(tid, 64 * WAVES);
    const size_t head = ((size_t)b.seq[i] * c.nkv + h) * c.nb;
    const bool has_dims = VD >= WAVES || wave * DT < VD;
    auto load = [](const i32x4* p) { return ONCE ? __builtin_nontemporal_load(p) : *p; };
    i32x4 kk[4][KD], vv[WAVES][DT];
    // a block's n-th kilobyte
    const uint32_t lane16 = lane * 16;
    auto kilo = [&](const int8_t* block, int n) { return load((const i32x4*)(block + n * 1024 + lane16)); };
    auto load_k = [&](int blk) {
        const int8_t* p = c.kc + (head + blk) * KV8_BLOCK * KR;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int d = 0; d < KD; ++d) kk[t][d] = kilo(p, t * KD + d);
    };
    auto load_v = [&](int base) {  // the wave's dims; a block behind the last: the last once more
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const int8_t* p = c.vc + (head + min(base + w, blk1 - 1)) * KV8_BLOCK * HD + wave * DT * 1024;
#pragma unroll
            for (int d = 0; d < DT; ++d) vv[w][d] = kilo(p, d);
        }
    };
    if (tile.blk0 + wave < blk1) load_k(tile.blk0 + wave);
    put_queries<HD, Wide>(tile, qs, qmax, lane, wave);
    const float qscale = 256.0f * query_scale<HD>(qmax[row]);
    const int pos = row < tile.rows ? tile.first + tile.token_of(row) : -1;
    const int from = a.window ? pos - a.window + 1 : 0;
    float m_run = -INFINITY, l_run = 0.0f;
    f32x4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int base = tile.blk0; base < blk1; base += WAVES) {
        const int blk = base + wave, blocks = min(blk1 - base, WAVES);
        if (has_dims) load_v(base);
        const float ks = scalar_load(c.ks + head + min(blk, blk1 - 1));
        float vs[WAVES];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) vs[w] = scalar_load(c.vs + head + min(base + w, blk1 - 1));
        float s[16], mb = -INFINITY, f = 0.0f;
        if (blk < blk1) {
            f = qscale * ks;
            f = f < 0x1p-126f ? 0x1p-126f : f;  // not zero: it meets -inf
            // The lowest digit's sum goes on top of the next one's, but for its
            // last 8 bits: an error below 2^-15 of q's largest magnitude times
            // one code, for all dims together, and much the same for all keys.
            i32x4 acc[4][3] = {};
            auto step = [&](int n, int d) {
                const i32x4 q = qs[n][d][lane];
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[t][n] = mfma(kk[t][d], q, acc[t][n]);
            };
#pragma unroll
            for (int n = 0; n < 3; ++n) {
#pragma unroll
                for (int t = 0; t < 4 && n == 1; ++t) acc[t][1] = acc[t][0] >> 8;
#pragma unroll
                for (int d = 0; d < KD; ++d) step(n, d);
            }
            if (blk + WAVES < blk1) load_k(blk + WAVES);
#pragma unroll
            for (int j = 0; j < 16; ++j) s[j] = (float)(acc[j / 4][2][j % 4] * 256 + acc[j / 4][1][j % 4]);
            if (tile.masked(blk)) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int p = blk * KV8_BLOCK + 16 * (j / 4) + 4 * g + j % 4;
                    s[j] = p <= pos && p >= from ? s[j] : -INFINITY;
                }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) mb = fmaxf(mb, s[j]);
            mb = fmaxf(mb, __shfl_xor(mb, 16, 64));
            mb = fmaxf(mb, __shfl_xor(mb, 32, 64));
            // nothing to see of the block: its scale, which may be NaN, has no say
            if (mb == -INFINITY) f = 1.0f;
            // in units of ln 2, and no less than any of them before its rounding
            mb *= f;
            mb = mb == -INFINITY ? mb : fmaf(fabsf(mb), 0x1p-23f, mb);
        }
        if (g == 0) st_m[wave][row] = mb;
        __syncthreads();
        // The row's maximum, and its largest scale of V: of the blocks that it
        // sees, whose values alone set what may be lost.  A scale that is NaN
        // is left out, and spoils the sums of the rows that see it instead.
        float ms = -INFINITY, top_vs = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float m = st_m[w][row];
            ms = fmaxf(ms, m);
            top_vs = fmaxf(top_vs, m != -INFINITY ? vs[w] : 0.0f);
        }
        // A row that sees nothing of the step has -inf for all its scores; one
        // whose scores are all NaN has the same maximum, and its sum becomes NaN.
        const float top = ms == -INFINITY ? 0.0f : ms;
        const float m_new = fmaxf(m_run, ms);
        const float alpha = m_run == m_new ? 1.0f : exp2_fast(m_run - m_new);
        const float beta = ms == -INFINITY ? 0.0f : exp2_fast(ms - m_new);
        m_run = m_new;
        if (blk < blk1) {
            const float mine = wave == 0 ? vs[0] : wave == 1 ? vs[1] : wave == 2 ? vs[2] : vs[3];
            const float share = mine == mine ? fminf(mine / fmaxf(top_vs, 0x1p-100f), 1.0f) * DIGIT_MAX : 0.0f;
            float lb = 0.0f;
            uint32_t pd[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float e = exp2_fast(fmaf(s[j], f, -top));
                lb += e;
                pd[j] = digits_of_share(e, share);
            }
            if (mine != mine && mb != -INFINITY) lb = mine;
            l_run = l_run * alpha + (ms == -INFINITY ? lb : lb * beta);
#pragma unroll
            for (int n = 0; n < 3; ++n) {
                i32x4 p;
#pragma unroll
                for (int t = 0; t < 4; ++t) p[t] = (int)(n < 2 ? byte_of(pd + 4 * t, n) ^ DIGIT_BIAS : byte_of(pd + 4 * t, n));
                ps[wave][n][lane] = p;
            }
        } else {
            l_run *= alpha;
        }
        __syncthreads();
        if (!has_dims) continue;
        i32x4 sum[DT][3];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            if (w >= blocks) break;
#pragma unroll
            for (int n = 0; n < 3; ++n) {
                const i32x4 p = ps[w][n][lane];
#pragma unroll
                for (int d = 0; d < DT; ++d) sum[d][n] = mfma(vv[w][d], p, w ? sum[d][n] : i32x4{0, 0, 0, 0});
            }
        }
        const float w = beta * top_vs * (1.0f / DIGIT_MAX);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[d][j] = fmaf(Wide::sum(sum[d][0][j], sum[d][1][j], sum[d][2][j]), w, o[d][j] * alpha);
    }
    // a row's sum: of its lanes, and of the waves' blocks
    l_run += __shfl_xor(l_run, 16, 64);
    l_run += __shfl_xor(l_run, 32, 64);
    if (g == 0) st_l[wave][row] = l_run;
    __syncthreads();
    if (row >= tile.rows || !has_dims) return;
    const float L = (st_l[0][row] + st_l[1][row]) + (st_l[2][row] + st_l[3][row]);
#pragma unroll
    for (int d = 0; d < DT; ++d) tile.put<HD>(row, 4 * (wave * DT + d) + g, o[d], m_run, L);
}

// Joins the chunk states of one output row: a workgroup takes 4 LN of its
// dims, its threads the chunks side by side, their outputs on the way before
// the weights are known.
template <int HD, int LN>
__global__ __launch_bounds__(NT) void k_kv8_combine(Kv8Batch b, Att8 a) {
    constexpr int GR = NT / LN, U = 4;  // groups that share the chunks, loads in flight
    __shared__ float red[8];
    __shared__ __align__(16) f32x4 sum[GR][LN];
    const int i = blockIdx.y, row = blockIdx.x / (HD / 4 / LN);
    if (row >= b.cnt[i] * a.heads) return;
    const size_t slot = (size_t)b.part[i] * a.heads + row;
    const int d4 = blockIdx.x % (HD / 4 / LN) * LN;
    const float* pm = a.part + slot * a.ns;
    const float* pl = a.part + (a.rows + slot) * a.ns;
    const f32x4* po = (const f32x4*)(a.part + 2 * a.rows * a.ns + slot * a.ns * HD) + d4;
    const int tid = threadIdx.x, ln = tid % LN, gr = tid / LN;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    // m and l of the thread's first chunk for the row's sums
    const float m0 = tid < a.ns ? pm[tid] : -INFINITY, l0 = tid < a.ns ? pl[tid] : 0.0f;
    f32x4 v[U];
    float mv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int j = min(gr + u * GR, a.ns - 1);
        v[u] = po[(size_t)j * (HD / 4) + ln];
        mv[u] = pm[j];
    }
    m = m0;
    for (int j = tid + NT; j < a.ns; j += NT) m = fmaxf(m, pm[j]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if ((tid & 63) == 0) red[tid >> 6] = m;
    __syncthreads();
    const float M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    auto weight = [&](float x) { return x == -INFINITY ? 0.0f : exp2_fast(x - M); };
    l = l0 * weight(m0);
    for (int j = tid + NT; j < a.ns; j += NT) l += pl[j] * weight(pm[j]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
    if ((tid & 63) == 0) red[4 + (tid >> 6)] = l;
    // a chunk that saw nothing wrote no output
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (gr + u * GR < a.ns && mv[u] != -INFINITY) acc += v[u] * weight(mv[u]);
    for (int j = gr + U * GR; j < a.ns; j += GR)
        if (pm[j] != -INFINITY) acc += po[(size_t)j * (HD / 4) + ln] * weight(pm[j]);
    sum[gr][ln] = acc;
    __syncthreads();
    if (tid < 4 * LN) {
        const float* t = (const float*)sum;
        const float L = (red[4] + red[5]) + (red[6] + red[7]);
        float r = 0.0f;
#pragma unroll
        for (int j = 0; j < GR; ++j) r += t[j * 4 * LN + tid];
        a.out[((size_t)b.off[i] * a.heads + row) * HD + 4 * d4 + tid] = r * (M == -INFINITY && L == 0.0f ? 0.0f : 1.0f / L);
    }
}

template <class F>
int with_hd(int hd, F&& f) {
    switch (hd) {
        case 32: f(std::integral_constant<int, 32>{}); break;
        case 64: f(std::integral_constant<int, 64>{}); break;
        case 128: f(std::integral_constant<int, 128>{}); break;
        case 256: f(std::integral_constant<int, 256>{}); break;
        default: return set_error(GH_ERR_INVALID, "unsupported head_dim %d", hd);
    }
    GH_HIP(hipGetLastError());
    return GH_OK;
}

}  // namespace

int launch_kv8_append(const Kv8Dev& c, int hd, const Kv8Batch& b, int n, int blocks, const float* k, const float* v,
                      hipStream_t s) {
    return with_hd(hd, [&](auto h) {
        hipLaunchKernelGGL(k_kv8_append<h.value>, dim3(blocks, 2 * c.nkv, n), dim3(4 * h.value), 0, s, c, b, k, v);
    });
}

int launch_kv8_truncate(const Kv8Dev& c, int hd, const Kv8Batch& b, int n, hipStream_t s) {
    return with_hd(hd, [&](auto h) {
        hipLaunchKernelGGL(k_kv8_truncate<h.value>, dim3(1, 2 * c.nkv, n), dim3(4 * h.value), 0, s, c, b);
    });
}

int launch_kv8_read(const Kv8Dev& c, int hd, const Kv8Batch& b, int n, int blocks, float* k, float* v, hipStream_t s) {
    return with_hd(hd, [&](auto h) {
        hipLaunchKernelGGL(k_kv8_read<h.value>, dim3(blocks, 2 * c.nkv, n), dim3(4 * h.value), 0, s, c, b, k, v);
    });
}

int launch_kv8_attention(const Kv8Dev& c, int hd, const Kv8Batch& b, int n, const Att8& a, hipStream_t s) {
    return with_hd(hd, [&](auto h) {
        if (a.tile == 4) hipLaunchKernelGGL((k_kv8_attention<h.value>), dim3(a.ns, c.nkv, n), dim3(64 * Narrow::WAVES), 0, s, c, b, a);
        else if (a.tiles == 1) hipLaunchKernelGGL((k_kv8_attention_wide<h.value, true>), dim3(a.ns * c.nkv, 1, n), dim3(64 * Wide::WAVES), 0, s, c, b, a);
        else hipLaunchKernelGGL((k_kv8_attention_wide<h.value, false>), dim3(a.ns * a.tiles * c.nkv, 1, n), dim3(64 * Wide::WAVES), 0, s, c, b, a);
        // few chunks: a row a workgroup (of 64 rows or more, so that they fill
        // the device): drafts of 16 sequences 31 us so, 32 by 32 dims
        constexpr int LN = h.value / 4;
        const unsigned rows = (unsigned)a.most_q * a.heads;
        if (a.ns > 1 && (a.ns > 4 * (NT / LN) || a.rows < 64)) hipLaunchKernelGGL((k_kv8_combine<h.value, 8>), dim3(rows * (h.value / 32), n), dim3(NT), 0, s, b, a);
        else if (a.ns > 1) hipLaunchKernelGGL((k_kv8_combine<h.value, LN>), dim3(rows, n), dim3(NT), 0, s, b, a);
    });
}

}  // namespace gh
