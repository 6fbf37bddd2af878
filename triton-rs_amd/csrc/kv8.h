// Key/value cache in 8 bits: layout, launch parameters and the launchers of kv8_cache.hip,
// kv8_few.hip and kv8_many.hip.
//
// A cache is num_pages pages of [Hkv][page_size / 16] blocks; a block holds 16 tokens of one head in
// 32 D + 16 bytes:
//   [0, 16 D)       keys: token t, dimension d at (d / 16) 256 + 16 t + d % 16
//   [16 D, 32 D)    values: token 4 quad + i, dimension r D / 16 + 4 g + e at g 1024 + quad 256 + 16 r + 4 e + i
//   [32 D, +16)     fp32 scale of the keys, of the values (powers of two); a 32-bit word, bit t: token t's key
//                   row is not finite, bit 16 + t: its value row; 4 bytes of zeros
// A byte is e4m3 (bias 7, 448 the largest, no infinities) and stands for itself times its scale; a row that is
// not finite has bytes of zero and its bit.
// The order is that of the matrix cores' operands: lane l of a wave takes the 16 bytes at 1024 x + 16 l, of keys
// 16 dimensions of token l % 16, of values four tokens of dimension l % 16 of four tiles.
#pragma once

#include "kv_attn.h"
#include "layer.h"

namespace w4a16 {

__host__ __device__ constexpr int kv8_block_bytes(int D) { return 32 * D + 16; }
constexpr int KV8_LEAST_EXP = -60;   // scales are 2^-60 at least

struct Kv8WriteParams {
    const void *k, *v;                // rows [T, Hkv, D], strides in elements
    int k_st, k_sh, v_st, v_sh;
    RopeRows q;                       // H = 0: none
    const int32_t* positions;         // [T], or null: a token's place in its sequence
    const double* inv_freq;           // null: no rotation
    float magnitude;                  // of keys,
    Magnitude q_magnitude;            // and for queries
    int rot;
    bool interleaved;
    unsigned char* cache;
    const int32_t *table, *kv_lens, *cu_q;
    int num_pages, pages_per_seq, T, B, Hkv, page_shift, max_q;
};
hipError_t launch_kv8_write(bool bf16, int D, const Kv8WriteParams& p, hipStream_t st);

struct Kv8ReadParams {
    void *k_out, *v_out;
    int k_st, k_sh, v_st, v_sh;
    const int32_t* slots;             // [T]; outside [0, num_pages * page_size): the row is passed over
    const unsigned char* cache;
    int num_pages, T, Hkv, page_shift;
};
hipError_t launch_kv8_read(bool bf16, int D, const Kv8ReadParams& p, hipStream_t st);

// Workgroups of kv8_few.hip that a compute unit has registers for, and those that the keys are split for: the four waves of one
// have enough of the cache on its way (D = 64: of two), and each further chunk costs its partial results' way. In us, for one, two,
// four a compute unit: 1 sequence, 8 heads of D = 128, 16000 keys 15.3, 16.7, 19.9; 16 of 16000 94.9, 99.3, 103.8; 8 of 3 queries, 2000
// keys 16.4, 17.5, 19.5; 4 of 16 heads of D = 64, 16000 keys 35.9, 30.8, 33.6.
constexpr int kv8_few_occupancy(int D, int nt) { return nt == 2 ? (D == 64 ? 3 : 2) : D <= 128 ? 4 : 2; }
constexpr int kv8_few_per_cu(int D) { return D == 64 ? 2 : 1; }
hipError_t launch_kv8_few(bool bf16, int D, const KvAttnParams& p, const KvAttnShape& s, hipStream_t st);
// Waves of kv8_many.hip a SIMD, by registers.
constexpr int kv8_many_simd_waves(int D, int groups) { return D <= 128 ? 2 : 1; }
hipError_t launch_kv8_many(bool bf16, int D, const KvAttnParams& p, const KvAttnShape& s, hipStream_t st);

}  // namespace w4a16
