// C-ABI entry points of the 8-bit key/value cache: argument checks (before any HIP call), then the
// launchers of kv8_cache.hip, kv8_few.hip and kv8_many.hip.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/w4a16.h"
#include "kv8.h"
#include "kv_api.h"

namespace w4a16 {

static bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }
static_assert(KV_COUNTER_BYTES == W4A16_KV8_COUNTER_BYTES, "counters fill their area");

constexpr int32_t KV8_MAX_TOKENS = 1 << 22;   // of a call that writes: their workgroups' threads are counted in 32 bits

// Keys in one chunk: 500 keys of one sequence, 8 heads of D = 128, 7.9 us whole, 9.3 in chunks, 1000 keys 10.5, 9.5; 4 drafts of 5
// tokens, 8 heads a group, 500 keys 13.1, 15.4.
constexpr int KV8_WHOLE_KEYS = 512;
// Up to this much a sequence's and head's last workgroup joins itself (us; itself, a kernel of its own): 1 sequence, 8 heads of
// D = 128, 31 chunks 13.2, 11.1; 5 queries of 8 heads a group, D = 256, 16 chunks of 40 KB 38.5, 25.1; 8 sequences of 3 queries, 4
// chunks of 6 KB 16.4, 17.2; 32 of 6, 24 KB in one 28.0, 34.0; 4 sequences, 8 chunks 36.3, 38.1.
constexpr int KV8_JOIN_CHUNKS = 12;
constexpr int64_t KV8_JOIN_BYTES = 96 << 10;
// One sequence alone, 8 heads of D = 128, takes 0.17 us for a step of 32 keys, 256 workgroups together 0.41: 16 sequences of 16000
// keys 123 us where a step alone is taken for 0.45 of the device's (whole), 95 from 0.55 to 0.7 (in two); 16 of 1000 keys 12.7
// up to 0.6 (whole), 14.1 at 0.7.
static const KvFormat KV8 = {"kv8 attention launch", [](int D, int) { return kv8_few_per_cu(D); }, kv8_many_simd_waves, KV8_WHOLE_KEYS,
                             [](int per_cu) { return 0.6f / (float)per_cu; }, 3.f, 8.f, KV8_JOIN_CHUNKS, KV8_JOIN_BYTES,
                             launch_kv8_few, launch_kv8_many};

}  // namespace w4a16

using namespace w4a16;

extern "C" {

W4A16_API size_t w4a16_kv8_cache_bytes(int32_t num_pages, int32_t Hkv, int32_t D, int32_t page_size) {
    if (num_pages < 1 || Hkv < 1 || Hkv > KV_MAX_HEADS || !kv_head_dim_ok(D) || !kv_page_ok(page_size) ||
        (int64_t)num_pages * page_size > INT32_MAX)
        return 0;
    return (size_t)num_pages * Hkv * (page_size / KV_BLOCK) * kv8_block_bytes(D);
}

W4A16_API int w4a16_kv8_write(void* stream, int elem, const void* k, int32_t k_stride_t, int32_t k_stride_h, const void* v,
                              int32_t v_stride_t, int32_t v_stride_h, const void* q, int32_t q_stride_t, int32_t q_stride_h,
                              void* q_out, int32_t qo_stride_t, int32_t qo_stride_h, const int32_t* positions,
                              const double* inv_freq, float magnitude, int32_t rot, int32_t interleaved, void* cache,
                              const int32_t* page_table, const int32_t* kv_lens, const int32_t* cu_q, int32_t T, int32_t B,
                              int32_t Hq, int32_t Hkv, int32_t D, int32_t num_pages, int32_t page_size,
                              int32_t pages_per_seq, int32_t max_q_len) {
    if (int rc = check_elem(elem)) return rc;
    if (int rc = check_geometry(num_pages, Hkv, D, page_size)) return rc;
    if (T < 0 || B < 0 || Hq < 0 || max_q_len < 1 || pages_per_seq < 1)
        return fail(W4A16_ERR_INVALID_ARG, "bad sizes (T=%d B=%d Hq=%d max_q_len=%d pages_per_seq=%d)", T, B, Hq, max_q_len, pages_per_seq);
    if (T > KV8_MAX_TOKENS) return fail(W4A16_ERR_UNSUPPORTED, "%d tokens: at most %d in a call", T, KV8_MAX_TOKENS);
    if (B > 65535) return fail(W4A16_ERR_UNSUPPORTED, "%d sequences: at most 65535 in a call", B);
    if (Hq > KV_MAX_HEADS) return fail(W4A16_ERR_UNSUPPORTED, "%d heads: at most %d", Hq, KV_MAX_HEADS);
    if (!cu_q && T != B) return fail(W4A16_ERR_INVALID_ARG, "without cu_q every sequence has one token (T=%d B=%d)", T, B);
    if (!cu_q && max_q_len != 1) return fail(W4A16_ERR_INVALID_ARG, "without cu_q max_q_len is 1, not %d", max_q_len);
    if (!q != (Hq == 0) || !q != !q_out) return fail(W4A16_ERR_INVALID_ARG, "q, q_out and Hq: all or none");
    if (!inv_freq && (q || positions)) return fail(W4A16_ERR_INVALID_ARG, "q and positions are for a rotation: inv_freq is null");
    if (inv_freq) {
        if (rot < 2 || rot % 2 || rot > D) return fail(W4A16_ERR_INVALID_ARG, "rot=%d: even, 2 to the head's %d dimensions", rot, D);
        if (!std::isfinite(magnitude)) return fail(W4A16_ERR_INVALID_ARG, "magnitude must be finite");
    }
    // (without sequences there are queries at most, at positions of their own)
    if (T == 0 || (B == 0 && (!q || !positions))) return W4A16_OK;
    if (!cache || (B > 0 && (!page_table || !kv_lens)))
        return fail(W4A16_ERR_INVALID_ARG, "null pointer argument (cache, page_table or kv_lens)");
    if (!aligned(cache, 16)) return fail(W4A16_ERR_INVALID_ARG, "cache must be 16-byte aligned");
    if (!aligned(page_table, 4) || !aligned(kv_lens, 4) || !aligned(cu_q, 4) || !aligned(positions, 4) || !aligned(inv_freq, 8))
        return fail(W4A16_ERR_INVALID_ARG, "page_table, kv_lens, cu_q and positions must be 4-byte aligned, inv_freq 8-byte");
    if (int rc = check_rows("k", k, k_stride_t, k_stride_h, T, Hkv, D, 8, false)) return rc;
    if (int rc = check_rows("v", v, v_stride_t, v_stride_h, T, Hkv, D, 8, false)) return rc;
    if (q) {
        if (int rc = check_rows("q", q, q_stride_t, q_stride_h, T, Hq, D, 1, false)) return rc;
        if (int rc = check_rows("q_out", q_out, qo_stride_t, qo_stride_h, T, Hq, D, 1, true)) return rc;
    }
    Kv8WriteParams p{};
    p.k = k; p.v = v; p.k_st = k_stride_t; p.k_sh = k_stride_h; p.v_st = v_stride_t; p.v_sh = v_stride_h;
    p.q = {q, q_out, q_stride_t, q_stride_h, qo_stride_t, qo_stride_h, Hq};
    p.positions = positions; p.inv_freq = inv_freq; p.magnitude = magnitude; p.q_magnitude = Magnitude::of(magnitude); p.rot = rot; p.interleaved = interleaved != 0;
    p.cache = static_cast<unsigned char*>(cache);
    p.table = page_table; p.kv_lens = kv_lens; p.cu_q = cu_q;
    p.num_pages = num_pages; p.pages_per_seq = pages_per_seq; p.T = T; p.B = B; p.Hkv = Hkv;
    p.page_shift = __builtin_ctz((unsigned)page_size); p.max_q = max_q_len;
    (void)hipGetLastError();
    const hipError_t e = launch_kv8_write(elem == W4A16_BF16, D, p, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? W4A16_OK : hip_fail(e, "kv8 write launch");
}

W4A16_API int w4a16_kv8_read(void* stream, int elem, const void* cache, const int32_t* slots, void* k_out, int32_t k_stride_t,
                             int32_t k_stride_h, void* v_out, int32_t v_stride_t, int32_t v_stride_h, int32_t num_pages,
                             int32_t T, int32_t Hkv, int32_t D, int32_t page_size) {
    if (int rc = check_elem(elem)) return rc;
    if (int rc = check_geometry(num_pages, Hkv, D, page_size)) return rc;
    if (T < 0) return fail(W4A16_ERR_INVALID_ARG, "T (%d) must not be negative", T);
    if (T > KV_MAX_ROWS) return fail(W4A16_ERR_UNSUPPORTED, "%d rows: at most %d in a call", T, KV_MAX_ROWS);
    if (T == 0) return W4A16_OK;
    if (!slots || !cache) return fail(W4A16_ERR_INVALID_ARG, "null pointer argument (slots or cache)");
    if (!aligned(cache, 16) || !aligned(slots, 4)) return fail(W4A16_ERR_INVALID_ARG, "cache must be 16-byte aligned, slots 4-byte");
    if (int rc = check_rows("k_out", k_out, k_stride_t, k_stride_h, T, Hkv, D, 8, true)) return rc;
    if (int rc = check_rows("v_out", v_out, v_stride_t, v_stride_h, T, Hkv, D, 8, true)) return rc;
    Kv8ReadParams p{};
    p.k_out = k_out; p.v_out = v_out; p.k_st = k_stride_t; p.k_sh = k_stride_h; p.v_st = v_stride_t; p.v_sh = v_stride_h;
    p.slots = slots; p.cache = static_cast<const unsigned char*>(cache);
    p.num_pages = num_pages; p.T = T; p.Hkv = Hkv; p.page_shift = __builtin_ctz((unsigned)page_size);
    (void)hipGetLastError();
    const hipError_t e = launch_kv8_read(elem == W4A16_BF16, D, p, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? W4A16_OK : hip_fail(e, "kv8 read launch");
}

W4A16_API size_t w4a16_kv8_attention_workspace_size(int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D,
                                                    int32_t max_q_len, int32_t max_kv_len) {
    return kv_attention_workspace_size(KV8, T, B, Hq, Hkv, D, max_q_len, max_kv_len);
}

// Which kernel a call runs, so that tests can hold a case to the path it is for; not part of the public header.
W4A16_API void w4a16_internal_kv8_path(int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_q_len,
                                       int32_t max_kv_len, int32_t* out) {
    kv_path(KV8, T, B, Hq, Hkv, D, max_q_len, max_kv_len, out);
}

W4A16_API int w4a16_kv8_attention(void* stream, int elem, const void* q, int32_t q_stride_t, int32_t q_stride_h,
                                  const void* cache, const int32_t* page_table, const int32_t* kv_lens,
                                  const int32_t* cu_q, void* out, int32_t out_stride_t, int32_t out_stride_h, float* lse,
                                  int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t num_pages,
                                  int32_t page_size, int32_t pages_per_seq, int32_t max_q_len, int32_t max_kv_len,
                                  float scale, int32_t causal, int32_t window, void* workspace, size_t workspace_bytes) {
    return kv_attention(KV8, stream, elem, q, q_stride_t, q_stride_h, cache, page_table, kv_lens, cu_q, out, out_stride_t,
                        out_stride_h, lse, T, B, Hq, Hkv, D, num_pages, page_size, pages_per_seq, max_q_len, max_kv_len, scale,
                        causal, window, workspace, workspace_bytes);
}

}  // extern "C"
