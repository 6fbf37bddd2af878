// C-ABI entry points of the 4-bit key/value cache: argument checks (before any HIP call), then the
// launchers of kv4_cache.hip, kv4_few.hip and kv4_many.hip.
#include <hip/hip_runtime.h>

#include "../../include/w4a16.h"
#include "kv4.h"
#include "kv_api.h"

namespace w4a16 {

static bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }
static_assert(KV_COUNTER_BYTES == W4A16_KV4_COUNTER_BYTES, "counters fill their area");

// Up to this much a sequence's and head's last workgroup joins itself; more is a kernel's, which costs its launch
// but waits for no counter. 32 queries' heads of 4096 keys, in us (itself, kernel): D = 128, 16 chunks 31.1, 20.1;
// 8 of 128 KB 28.3, 26.5; 5 of 84 KB 32.6, 33.1. 8 heads: 16 chunks 22.6, 19.1; 10 chunks 21.4, 23.3; 4 35.2, 38.4.
constexpr int KV4_JOIN_CHUNKS = 12;
constexpr int64_t KV4_JOIN_BYTES = 96 << 10;
static const KvFormat KV4 = {"kv4 attention launch", kv4_few_per_cu, kv4_many_simd_waves, KV4_WHOLE_KEYS, [](int) { return 0.45f; }, 6.f, 7.f,
                             KV4_JOIN_CHUNKS, KV4_JOIN_BYTES, launch_kv4_few, launch_kv4_many};

static int kv4_rows(bool write, void* stream, int elem, void* k, void* v, int32_t k_st, int32_t k_sh, int32_t v_st,
                    int32_t v_sh, const int32_t* slots, void* cache, int32_t num_pages, int32_t T, int32_t Hkv,
                    int32_t D, int32_t page_size) {
    if (int rc = check_elem(elem)) return rc;
    if (int rc = check_geometry(num_pages, Hkv, D, page_size)) return rc;
    if (T < 0) return fail(W4A16_ERR_INVALID_ARG, "T (%d) must not be negative", T);
    if (T > KV_MAX_ROWS) return fail(W4A16_ERR_UNSUPPORTED, "%d rows: at most %d in a call", T, KV_MAX_ROWS);
    if (T == 0) return W4A16_OK;
    if (!slots || !cache) return fail(W4A16_ERR_INVALID_ARG, "null pointer argument (slots or cache)");
    if (!aligned(cache, 16) || !aligned(slots, 4)) return fail(W4A16_ERR_INVALID_ARG, "cache must be 16-byte aligned, slots 4-byte");
    if (int rc = check_rows(write ? "k" : "k_out", k, k_st, k_sh, T, Hkv, D, 8, !write)) return rc;
    if (int rc = check_rows(write ? "v" : "v_out", v, v_st, v_sh, T, Hkv, D, 8, !write)) return rc;
    Kv4RowParams p{};
    p.k = p.k_out = k; p.v = p.v_out = v;
    p.k_st = k_st; p.k_sh = k_sh; p.v_st = v_st; p.v_sh = v_sh;
    p.slots = slots; p.cache = static_cast<unsigned char*>(cache);
    p.num_pages = num_pages; p.T = T; p.Hkv = Hkv; p.page_shift = __builtin_ctz((unsigned)page_size);
    hipStream_t st = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    const hipError_t e = write ? launch_kv4_write(elem == W4A16_BF16, D, p, st) : launch_kv4_read(elem == W4A16_BF16, D, p, st);
    return e == hipSuccess ? W4A16_OK : hip_fail(e, write ? "kv4 write launch" : "kv4 read launch");
}

}  // namespace w4a16

using namespace w4a16;

extern "C" {

W4A16_API size_t w4a16_kv4_cache_bytes(int32_t num_pages, int32_t Hkv, int32_t D, int32_t page_size) {
    if (num_pages < 1 || Hkv < 1 || Hkv > KV_MAX_HEADS || !kv_head_dim_ok(D) || !kv_page_ok(page_size) ||
        (int64_t)num_pages * page_size > INT32_MAX)
        return 0;
    return (size_t)num_pages * Hkv * (page_size / KV_BLOCK) * kv4_block_bytes(D);
}

W4A16_API int w4a16_kv4_write(void* stream, int elem, const void* k, const void* v, int32_t k_stride_t,
                              int32_t k_stride_h, int32_t v_stride_t, int32_t v_stride_h, const int32_t* slots,
                              void* cache, int32_t num_pages, int32_t T, int32_t Hkv, int32_t D, int32_t page_size) {
    return kv4_rows(true, stream, elem, const_cast<void*>(k), const_cast<void*>(v), k_stride_t, k_stride_h, v_stride_t,
                    v_stride_h, slots, cache, num_pages, T, Hkv, D, page_size);
}

W4A16_API int w4a16_kv4_read(void* stream, int elem, const void* cache, const int32_t* slots, void* k_out, void* v_out,
                             int32_t k_stride_t, int32_t k_stride_h, int32_t v_stride_t, int32_t v_stride_h,
                             int32_t num_pages, int32_t T, int32_t Hkv, int32_t D, int32_t page_size) {
    return kv4_rows(false, stream, elem, k_out, v_out, k_stride_t, k_stride_h, v_stride_t, v_stride_h, slots,
                    const_cast<void*>(cache), num_pages, T, Hkv, D, page_size);
}

W4A16_API size_t w4a16_kv4_attention_workspace_size(int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D,
                                                    int32_t max_q_len, int32_t max_kv_len) {
    return kv_attention_workspace_size(KV4, T, B, Hq, Hkv, D, max_q_len, max_kv_len);
}

// Which kernel a call runs, so that tests can hold a case to the path it is for; not part of the public header.
W4A16_API void w4a16_internal_kv4_path(int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_q_len,
                                       int32_t max_kv_len, int32_t* out) {
    kv_path(KV4, T, B, Hq, Hkv, D, max_q_len, max_kv_len, out);
}

W4A16_API int w4a16_kv4_attention(void* stream, int elem, const void* q, int32_t q_stride_t, int32_t q_stride_h,
                                  const void* cache, const int32_t* page_table, const int32_t* kv_lens,
                                  const int32_t* cu_q, void* out, int32_t out_stride_t, int32_t out_stride_h, float* lse,
                                  int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t num_pages,
                                  int32_t page_size, int32_t pages_per_seq, int32_t max_q_len, int32_t max_kv_len,
                                  float scale, int32_t causal, int32_t window, void* workspace, size_t workspace_bytes) {
    return kv_attention(KV4, stream, elem, q, q_stride_t, q_stride_h, cache, page_table, kv_lens, cu_q, out, out_stride_t,
                        out_stride_h, lse, T, B, Hq, Hkv, D, num_pages, page_size, pages_per_seq, max_q_len, max_kv_len, scale,
                        causal, window, workspace, workspace_bytes);
}

}  // extern "C"
