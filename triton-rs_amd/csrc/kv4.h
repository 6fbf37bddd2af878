// Key/value cache in 4 bits: layout, launch parameters and the launchers of kv4_cache.hip,
// kv4_few.hip and kv4_many.hip.
//
// A cache is num_pages pages of [Hkv][page_size / 16] blocks; a block holds 16 tokens of one head in
// 16 D + 128 bytes:
//   [0, 8 D)        keys: row `tok` at tok D / 2, dimension d in nibble d of the row (lowest first)
//   [8 D, 16 D)     values: token tok = 4 quad + 2 pair + i, dimension d = column D / 16 + 4 h + e in
//                   nibble e of the 16-bit word at quad 2 D + column D / 8 + pair D / 16 + 4 h + 2 i
//   [16 D, +64)     keys' parameters, one 32-bit word a token: scale (bits 0..15, the element
//                   type's bits), zero point 0..15 (bits 16..31), as in the prepared weights' table
//   [16 D + 64, +64) values' parameters
// A nibble n stands for (n - zero) * scale, exact in fp32.
// The order serves the matrix cores: a lane of an MFMA operand takes consecutive k of one row. With
// keys the k are dimensions, so a row's nibbles lie together; with values they are tokens, so two
// tokens share a 32-bit word, in its two halves, where one mask turns them into a pair of operands.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace w4a16 {

constexpr int KV4_BLOCK = 16;   // tokens of a block
__host__ __device__ constexpr int kv4_block_bytes(int D) { return 16 * D + 128; }
constexpr bool kv4_head_dim_ok(int D) { return D == 64 || D == 128 || D == 192 || D == 256; }
constexpr bool kv4_page_ok(int P) { return P >= 16 && P <= 1024 && (P & (P - 1)) == 0; }

struct Kv4RowParams {
    const void *k, *v;                // write: rows [T, Hkv, D], strides in elements
    void *k_out, *v_out;              // read
    int k_st, k_sh, v_st, v_sh;
    const int32_t* slots;             // [T]; outside [0, num_pages * page_size): the row is passed over
    unsigned char* cache;
    int num_pages, T, Hkv, page_shift;   // page_size = 1 << page_shift
};
hipError_t launch_kv4_write(bool bf16, int D, const Kv4RowParams& p, hipStream_t st);
hipError_t launch_kv4_read(bool bf16, int D, const Kv4RowParams& p, hipStream_t st);

struct Kv4AttnParams {
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
    int causal, window;
    uint32_t* counters;               // kv4_few.hip: one a sequence, head and tile, zero between calls
    float* partials;                  // by number of chunk, slot_cols (D + 2) floats each
    // from the shape
    int G, slot_cols;
    int tiles, splits, chunk, pair_tiles, rows;  // kv4_many.hip
    int places, budget, at_once, whole, join_apart, join_parts;   // kv4_few.hip
};
constexpr size_t KV4_MAX_COUNTERS = 16384;
struct Kv4AttnShape {
    bool many;         // kv4_many.hip, else kv4_few.hip
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
    int few_q;         // many: sequences of up to this many queries go to kv4_few.hip first (0: none do)
};
// Workgroups of kv4_few.hip that are planned for a compute unit: what registers (90, 130; 123, 187; 157; 190 of D = 64, 128,
// 192, 256 with one and, up to 128, two column tiles a wave) and LDS leave room for, one less at D = 64 with one tile.
constexpr int kv4_few_per_cu(int D, int nt) { return nt == 2 ? (D == 64 ? 3 : 2) : D <= 128 ? 4 : D == 192 ? 3 : 2; }
constexpr int KV4_WHOLE_KEYS = 512;   // keys that kv4_few.hip leaves in one chunk
hipError_t launch_kv4_few(bool bf16, int D, const Kv4AttnParams& p, const Kv4AttnShape& s, hipStream_t st);
// Waves of kv4_many.hip a SIMD, by registers (144, 213, 376 and 485 of D = 64, 128, 192 and 256).
constexpr int kv4_many_simd_waves(int D, int groups) { return D == 64 && groups == 1 ? 3 : D <= 128 ? 2 : 1; }
hipError_t launch_kv4_many(bool bf16, int D, const Kv4AttnParams& p, const Kv4AttnShape& s, hipStream_t st);

}  // namespace w4a16
