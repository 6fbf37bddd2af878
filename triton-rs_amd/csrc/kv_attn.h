// Attention over a paged key/value cache in fewer bits: launch parameters and plan, the same for the caches
// in 4 bits (kv4.h) and in 8 (kv8.h). A cache is num_pages pages of [Hkv][page_size / 16] blocks of 16 tokens of
// one head, in as many bytes as its format takes.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace w4a16 {

constexpr int KV_BLOCK = 16;   // tokens of a block
constexpr bool kv_head_dim_ok(int D) { return D == 64 || D == 128 || D == 192 || D == 256; }
constexpr bool kv_page_ok(int P) { return P >= 16 && P <= 1024 && (P & (P - 1)) == 0; }

struct KvAttnParams {
    const void* q;                    // [T, Hq, D]
    void* out;                        // [T, Hq, D]
    float* lse;                       // [T, Hq] or null
    const unsigned char* cache;
    const int32_t* table;             // [B, pages_per_seq]
    const int32_t* kv_lens;           // [B]
    const int32_t* cu_q;              // [B + 1], or null: one query a sequence
    int q_st, q_sh, o_st, o_sh;
    int num_pages, pages_per_seq, T, B, Hq, Hkv, page_shift, max_q, max_kv;
    int least_q, most_q;              // sequences of fewer or more queries are another kernel's
    float scale_mant;                 // scale * log2(e) = scale_mant 2^scale_exp, |scale_mant| < 1
    int scale_exp;
    float scale_log2;                 // scale * log2(e)
    int causal, window;
    uint32_t* counters;               // few columns: one a sequence, head and tile, zero between calls
    float* partials;                  // by number of chunk, slot_cols (D + 2) floats each
    // from the shape
    int G, slot_cols;
    int tiles, splits, chunk, pair_tiles, rows;  // many columns
    int places, budget, at_once, whole, join_apart, join_parts;   // few columns
    int whole_keys;                   // few columns: a sequence of up to so many keys is one chunk
    float step_alone, round_cost, join_cost;   // few columns: in steps of a full device (kv_few.h)
};
constexpr size_t KV_MAX_COUNTERS = 16384;
struct KvAttnShape {
    bool many;         // the kernel for many columns, else that for few
    int nt;            // columns of a wave / 16
    int tiles;         // tiles of columns of a sequence and key/value head
    int slot_cols;     // columns of a chunk's partial results
    // many: groups of four waves a workgroup; chunks of the keys, at most, and their length; long and short tiles of
    // columns by turns; tiles of all sequences of a head, at most (0: every sequence has a row of `tiles`)
    int groups, splits, chunk, rows;
    bool pair_tiles;
    // few: chunks of all sequences of a head, at most, about how many are wanted, and how many run at once; whole: one a sequence;
    // join_apart: chunks are joined by a kernel of their own
    int places, budget, at_once;
    bool whole, join_apart;
    size_t partial_bytes;
    int few_q;         // many: sequences of up to this many queries go to the kernel for few first (0: none do)
};

}  // namespace w4a16
