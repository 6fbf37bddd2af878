// Internal host-side interface of kv_api.cpp: what the entry points of the caches in 4 and in 8 bits share.
#pragma once

#include "kv_attn.h"
#include "launch.h"

namespace w4a16 {

constexpr int KV_MAX_HEADS = 1024;
constexpr int KV_MAX_ROWS = 1 << 27;   // rows of one call: 16 threads each of a 32-bit count of threads
constexpr size_t KV_COUNTER_BYTES = KV_MAX_COUNTERS * sizeof(uint32_t);

// What attention's plan has to know of a cache's format, and its kernels.
struct KvFormat {
    const char* name;
    int (*few_per_cu)(int D, int nt);           // workgroups of the kernel for few columns that a compute unit holds
    int (*many_simd_waves)(int D, int groups);  // waves of the kernel for many columns that a SIMD holds
    int whole_keys;                             // keys that the kernel for few columns leaves in one chunk
    float (*step_alone)(int per_cu);            // in steps of a full device (kv_few.h), as
    float round_cost, join_cost;                // these
    int join_chunks;                            // up to this much a sequence's and head's last workgroup joins itself
    int64_t join_bytes;
    hipError_t (*launch_few)(bool bf16, int D, const KvAttnParams& p, const KvAttnShape& s, hipStream_t st);
    hipError_t (*launch_many)(bool bf16, int D, const KvAttnParams& p, const KvAttnShape& s, hipStream_t st);
};

// Status codes, with the calling thread's message set where they are errors.
int check_elem(int elem);
int check_geometry(int32_t num_pages, int32_t Hkv, int32_t D, int32_t page_size);
// Rows [T, H, D] of 16-bit elements at these strides (elements), D contiguous: all multiples of `unit` elements, and for
// an output no two rows over each other.
int check_rows(const char* what, const void* p, int32_t st, int32_t sh, int32_t T, int32_t H, int32_t D, int unit, bool out);

size_t kv_attention_workspace_size(const KvFormat& f, int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D,
                                   int32_t max_q_len, int32_t max_kv_len);
// Which kernel a call runs. out: {1, column tiles a wave, chunks a head at most, joined by a kernel of their own} few
// columns; {2, wave groups, chunks, queries of sequences that run on the other (0: none do)} many.
void kv_path(const KvFormat& f, int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_q_len, int32_t max_kv_len, int32_t* out);
int kv_attention(const KvFormat& f, void* stream, int elem, const void* q, int32_t q_stride_t, int32_t q_stride_h,
                 const void* cache, const int32_t* page_table, const int32_t* kv_lens, const int32_t* cu_q, void* out,
                 int32_t out_stride_t, int32_t out_stride_h, float* lse, int32_t T, int32_t B, int32_t Hq, int32_t Hkv,
                 int32_t D, int32_t num_pages, int32_t page_size, int32_t pages_per_seq, int32_t max_q_len,
                 int32_t max_kv_len, float scale, int32_t causal, int32_t window, void* workspace, size_t workspace_bytes);

}  // namespace w4a16
