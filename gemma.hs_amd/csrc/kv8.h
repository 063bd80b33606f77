// The 8-bit KV cache of a batch: handle, device layout and launchers.
#pragma once

#include "common.h"

struct gh_kv8 {
    gh_ctx* ctx = nullptr;
    int n_seq = 0, max_seq = 0, nkv = 0, hd = 0;
    int nb = 0;                 // blocks a sequence
    std::vector<int32_t> len;   // tokens a sequence (host)
    std::vector<int32_t> mark;  // per sequence: the call that named it last (no sequence twice)
    int32_t call = 0;
    void* mem = nullptr;  // the one allocation that holds everything below
    int8_t *kc = nullptr, *vc = nullptr;
    float *ks = nullptr, *vs = nullptr;
    float *kt = nullptr, *vt = nullptr;
    ~gh_kv8();
};

namespace gh {

constexpr int KV8_BLOCK = GH_KV8_BLOCK;

// Codes of a block lie in the order in which a wave's lanes feed them to the
// 16x16x64 int8 matrix instruction, 16 bytes a lane, so that every load of
// the attention is 1 KB of consecutive bytes and its probabilities need no
// shuffle.  With g = lane / 16, r = lane % 16:
//   K  [token / 16][dim / 64][lane][byte]   token 16 t + r, dim 64 c + 16 g + byte
//   V  [dim / 16][lane][byte]               dim 16 c + r, byte 4 t + i: token 16 t + 4 g + i
// K rows of 32 dims are padded to 64 (the padding meets query digits of zero).
// kc [n_seq][nkv][nb][64 * max(hd, 64)], vc [n_seq][nkv][nb][64 * hd],
// ks, vs [n_seq][nkv][nb], kt, vt [n_seq][nkv][64][hd]: the f32 rows of the
// partly filled last block.
constexpr int kv8_k_row(int hd) { return hd < 64 ? 64 : hd; }

struct Kv8Dev {
    int8_t *kc, *vc;
    float *ks, *vs;
    float *kt, *vt;
    int nkv, nb;
};

// Up to KV8_BATCH sequences of a call, by value in a kernel's arguments (no
// copy to the device, and the host has checked every number).
constexpr int KV8_BATCH = 192;
struct Kv8Batch {
    int seq[KV8_BATCH];
    int pos[KV8_BATCH];   // append, truncate: tokens before; read: begin; attention: tokens
    int off[KV8_BATCH];   // first of the entry's rows among the call's
    int cnt[KV8_BATCH];   // new tokens; tokens to read; query tokens; truncate: the new length itself
    int part[KV8_BATCH];  // attention: first of the entry's query tokens among the launch's
};

// blocks: the most that one of the entries touches
int launch_kv8_append(const Kv8Dev& c, int hd, const Kv8Batch& b, int n, int blocks, const float* k, const float* v,
                      hipStream_t s);
int launch_kv8_truncate(const Kv8Dev& c, int hd, const Kv8Batch& b, int n, hipStream_t s);
int launch_kv8_read(const Kv8Dev& c, int hd, const Kv8Batch& b, int n, int blocks, float* k, float* v, hipStream_t s);

// Query rows of a kv head are (token, head of its group) pairs, 4 or 16 of them
// a tile.
struct Att8 {
    const float* q;
    float* out;
    float* part;  // chunk states: m [rows][ns], l [rows][ns], o [rows][ns][hd]; rows = heads * query tokens
    size_t rows;
    int most_q;          // query tokens of the entry that has most
    int heads, group;    // query heads, per kv head
    unsigned group_inv;  // ceil(2^32 / group): the upper half of row * group_inv is row / group (0 for group 1)
    int window;
    int tile;   // rows a tile
    int tiles;  // row tiles of the longest entry
    int ns;     // key chunks of the longest entry
    int chunk;  // blocks a chunk at most: an entry's chunks are of one size
};
int launch_kv8_attention(const Kv8Dev& c, int hd, const Kv8Batch& b, int n, const Att8& a, hipStream_t s);

}  // namespace gh
