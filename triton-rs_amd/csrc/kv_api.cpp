// Attention over a paged key/value cache, the part of its C-ABI entry points that both formats (kv4_api.cpp,
// kv8_api.cpp) share: argument checks (before any HIP call), the choice of a kernel and the split of the keys.
#include "kv_api.h"

#include <algorithm>
#include <cmath>

#include "../../include/w4a16.h"

namespace w4a16 {

static bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

// Compute units that the split of the keys is planned for: MI355X's, so that a workspace's size is the same wherever it is asked for.
constexpr int KV_CUS = 256;
constexpr int KV_MAX_KEYS = 1 << 30;   // of a sequence: positions a few steps further still are int32
constexpr int64_t KV_MAX_ALL_KEYS = 1ll << 36;   // of all sequences: their steps of 32 are summed in 32 bits
constexpr int64_t KV_MAX_SPLIT_TILES = 4096;   // of 128 columns, 66 KB of partial results (D = 128) a chunk each

int check_elem(int elem) {
    if (elem != 0 && elem != W4A16_BF16) return fail(W4A16_ERR_INVALID_ARG, "unknown element type %d", elem);
    return W4A16_OK;
}

int check_geometry(int32_t num_pages, int32_t Hkv, int32_t D, int32_t page_size) {
    if (num_pages < 1 || Hkv < 1 || D < 1 || page_size < 1)
        return fail(W4A16_ERR_INVALID_ARG, "sizes must be positive (num_pages=%d Hkv=%d D=%d page_size=%d)", num_pages,
                    Hkv, D, page_size);
    if (!kv_head_dim_ok(D)) return fail(W4A16_ERR_UNSUPPORTED, "head dimension %d: 64, 128, 192 or 256", D);
    if (!kv_page_ok(page_size)) return fail(W4A16_ERR_UNSUPPORTED, "page_size %d: a power of two from 16 to 1024", page_size);
    if (Hkv > KV_MAX_HEADS) return fail(W4A16_ERR_UNSUPPORTED, "%d heads: at most %d", Hkv, KV_MAX_HEADS);
    if ((int64_t)num_pages * page_size > INT32_MAX)
        return fail(W4A16_ERR_UNSUPPORTED, "%d pages of %d tokens: slots are int32", num_pages, page_size);
    return W4A16_OK;
}

int check_rows(const char* what, const void* p, int32_t st, int32_t sh, int32_t T, int32_t H, int32_t D, int unit, bool out) {
    if (!p) return fail(W4A16_ERR_INVALID_ARG, "null pointer argument (%s)", what);
    if (!aligned(p, 2 * unit)) return fail(W4A16_ERR_INVALID_ARG, "%s must be %d-byte aligned", what, 2 * unit);
    if (st < 0 || sh < 0 || st % unit || sh % unit)
        return fail(W4A16_ERR_INVALID_ARG, "%s: strides (%d, %d) must be non-negative multiples of %d elements", what, st, sh, unit);
    if (out) {
        const bool token_major = (H == 1 || sh >= D) && (T == 1 || st >= (int64_t)(H - 1) * sh + D);
        const bool head_major = (T == 1 || st >= D) && (H == 1 || sh >= (int64_t)(T - 1) * st + D);
        if (!token_major && !head_major)
            return fail(W4A16_ERR_INVALID_ARG, "%s: rows at strides (%d, %d) lie over each other", what, st, sh);
    }
    return W4A16_OK;
}

// Which kernel, and how the keys are split, by one set of rules for both caches. They were set by the times in 4 bits that stand
// first; those in 8 bits (captured, the same keys each time) stand beside them, also where the rule loses.
//
// Few columns (up to 64) go to the kernel whose waves share them: 8 sequences
// of 8 queries, 8 heads of 4096 keys, D = 128, 64 columns, 37.5 us against 43.9 on the other, 96 columns 56.7 against
// 45.5. (8 bits: 64 columns 37.2, 36.6, 80 columns 54.4, 38.3; D = 64 25.7, 27.3 and 62.7, 28.1; D = 256 53.8, 79.7 and 80.1, 81.1. One
// sequence alone would do better on it up to 128 columns and more: 19.9, 26.3, at D = 256 25.8, 46.8.)
// Its waves take two tiles of 16 columns from 17 on (32 sequences, 24 columns: 46.9 us, one tile 65.0; 8 bits 46.5, 56.5, of 8 sequences
// 24.6, 24.9, of one 14.3, 12.9), where registers allow (D <= 128). The keys are split as far as it takes to fill the places of
// workgroups that run at once, no further: each chunk costs its partial results a round trip through memory.
static KvAttnShape kv_attention_shape(const KvFormat& f, int T, int B, int Hq, int Hkv, int D, int max_q, int max_kv) {
    KvAttnShape s{};
    const int64_t G = Hq / Hkv, C = (int64_t)(max_q < T ? max_q : T) * G, slots_of_cu = KV_CUS;
    s.many = C > 64;
    s.nt = s.many || (C > 16 && D <= 128) ? 2 : 1;
    const int wg_cols = s.many ? 128 : 32 * s.nt;
    const int64_t tiles = std::max<int64_t>(1, (C + wg_cols - 1) / wg_cols);
    int64_t items = std::max<int64_t>(1, tiles * B * Hkv);
    s.tiles = (int)std::min<int64_t>(tiles, 1 << 30);
    size_t slots = 0;
    // Few rows for what the sequences may have: single tokens among prompts. Walking a long cache for 128 columns of which
    // few are there holds up the rest (31 single tokens and a chunk of 1024, 4096 keys each, 32 heads on 8, D = 128: 382 us
    // on the kernel for many columns alone, 181 on both; 139 in a call each, where the chunk's tiles are counted alone and split).
    // (In 8 bits a loss: 134 alone, 156 on both; 7 single tokens and a chunk of 512, 2048 keys each, 44 and 60, 3 of them 43.4 and 43.5.)
    const int few_q = (int)(64 / G);
    s.few_q = s.many && B > 1 && few_q > 0 && 4 * (int64_t)T < (int64_t)B * max_q ? few_q : 0;
    if (s.many) {
        // Up to 1024 sequences share one row of tiles where that is less than half of as many as the longest has for each:
        // no more tiles than T rows of q make. (Finding its own costs a workgroup a microsecond.)
        const int64_t rows = std::max<int64_t>(1, (T * G + 127 * (int64_t)B) / 128);
        int64_t full = items;   // about as many as there are
        if (B > 1 && B <= 1024 && 2 * rows < tiles * B && rows <= 65535) {
            // (launched: those of sequences that run here, which have a query at least, or more than few_q)
            s.rows = (int)std::max<int64_t>(1, (T * G + 127 * std::min<int64_t>(B, T / (s.few_q + 1))) / 128);
            items = rows * Hkv;
            full = std::max<int64_t>(1, (T * G + 127) / 128 * Hkv);
        }
        // Up to two tiles a compute unit: two groups of waves share a tile's keys (a prompt of
        // 2048, 32 heads: 64 us, one group 75; 1344 tiles of 7 prompts: 58, one 45; 8 bits 60, 65 and, prompts of 50 to 1500 tokens, 16 heads of
        // 64, 54, one 43). Not where the tiles are of one length (a chunk behind a long context) and fill the device by themselves (1024
        // over 32768: 670, one 664, before the reference followed the value scales; 8 bits 613, one 629).
        s.groups = D <= 128 && full <= 2 * KV_CUS && !(full >= KV_CUS && max_kv >= 2 * (int64_t)max_q) ? 2 : 1;
        const int64_t at_once = slots_of_cu * f.many_simd_waves(D, s.groups) / s.groups;
        // Chunks of 512 keys or more (64 queries over 4096 keys, 32 heads on 8 of D = 128, 30.5 us so, of 256 34.3, of 1024
        // 36.3; over 2048 26.0, 25.4, 34.4; 8 bits 28.0, 33.5, 31.5 and 23.7, 24.2, 30.0, but 16 heads on 2 of D = 256 over 2048 keys 42.9, of
        // 256 35.7, over 512 36.3, of 128 25.6), as many as run at once: a last round for a few workgroups costs as much as a full
        // one (154 queries of 24 heads on one over 18208 keys, 29 tiles in 9 chunks, 2 rounds, 112.5 us, in 8 69.4).
        int64_t most = std::max<int64_t>(1, std::min(at_once / full, ((int64_t)max_kv + 511) / 512));
        if (items > KV_MAX_SPLIT_TILES) most = 1;
        s.chunk = (int)std::max<int64_t>(128, (((int64_t)max_kv + most - 1) / most + 127) / 128 * 128);
        s.splits = std::max(1, (int)(((int64_t)max_kv + s.chunk - 1) / s.chunk));
        s.pair_tiles = full * s.splits <= at_once;
        s.slot_cols = wg_cols;
        if (most > 1) slots = (size_t)items * most;   // (which grows with max_kv, and splits are no more: enough for a smaller one, too)
    } else {
        // chunks of a head and tile: what runs at once, or several rounds of it; B sequences have one each at least,
        // and a remainder
        const int64_t at_once = std::max<int64_t>(1, slots_of_cu * f.few_per_cu(D, s.nt) / (Hkv * tiles));
        const int64_t rounds = (2 * (int64_t)B + at_once - 1) / at_once;
        s.whole = items > (int64_t)KV_MAX_COUNTERS || max_kv <= f.whole_keys;
        // up to 128 of a sequence, as many as one join takes in its time (131072 keys of one head: 1024 chunks 47.6 us)
        s.budget = (int)std::max<int64_t>(2 * (int64_t)B, std::min<int64_t>(rounds * at_once, 128 * (int64_t)B));
        s.at_once = (int)at_once;
        s.places = (int)(s.whole ? B : std::min<int64_t>(s.budget, (int64_t)B * (((int64_t)max_kv + 31) / 128 + 1)));
        s.slot_cols = (int)std::min<int64_t>(wg_cols, (C + 15) / 16 * 16);
        if (!s.whole) slots = (size_t)tiles * Hkv * s.places;
        // the chunks of a sequence, in a batch of like ones
        const int64_t chunks = std::min<int64_t>(s.budget / std::max(B, 1), ((int64_t)max_kv + 127) / 128);
        s.join_apart = !s.whole && (chunks > f.join_chunks || C * D * 4 * chunks >= f.join_bytes);
    }
    s.partial_bytes = slots * s.slot_cols * (D + 2) * sizeof(float);
    return s;
}
// The part of such a batch that runs on the kernel for few columns.
static KvAttnShape kv_few_part(const KvFormat& f, const KvAttnShape& s, int T, int B, int Hq, int Hkv, int D, int max_kv) {
    return kv_attention_shape(f, T, B, Hq, Hkv, D, s.few_q, max_kv);
}
// Workspace beyond the counters.
static size_t kv_partial_bytes(const KvFormat& f, const KvAttnShape& s, int T, int B, int Hq, int Hkv, int D, int max_kv) {
    return s.partial_bytes + (s.few_q ? kv_few_part(f, s, T, B, Hq, Hkv, D, max_kv).partial_bytes : 0);
}
static void kv_params(const KvFormat& f, KvAttnParams& p, const KvAttnShape& s, int D, int max_q, int T) {
    p.max_q = max_q < T ? max_q : T;
    p.slot_cols = s.slot_cols;
    p.whole_keys = f.whole_keys; p.step_alone = f.step_alone(f.few_per_cu(D, s.nt)); p.round_cost = f.round_cost; p.join_cost = f.join_cost;
    p.rows = s.rows; p.tiles = s.tiles; p.splits = s.splits; p.chunk = s.chunk; p.pair_tiles = s.pair_tiles;
    p.places = s.places; p.budget = s.budget; p.at_once = s.at_once; p.whole = s.whole; p.join_apart = s.join_apart;
    p.join_parts = (int)((std::min<int64_t>((int64_t)p.max_q * p.G, 32 * s.nt) * (D / 4) + 63) / 64);
}

static int check_attention(const KvFormat& f, int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_q, int32_t max_kv) {
    if (T < 0 || B < 0 || max_q < 1 || max_kv < 0)
        return fail(W4A16_ERR_INVALID_ARG, "bad sizes (T=%d B=%d max_q_len=%d max_kv_len=%d)", T, B, max_q, max_kv);
    if (Hq < 1 || Hkv < 1 || Hq % Hkv)
        return fail(W4A16_ERR_INVALID_ARG, "%d query heads must be a multiple of %d key/value heads", Hq, Hkv);
    if (!kv_head_dim_ok(D)) return fail(W4A16_ERR_UNSUPPORTED, "head dimension %d: 64, 128, 192 or 256", D);
    if (Hq > KV_MAX_HEADS) return fail(W4A16_ERR_UNSUPPORTED, "%d heads: at most %d", Hq, KV_MAX_HEADS);
    if (max_kv > KV_MAX_KEYS) return fail(W4A16_ERR_UNSUPPORTED, "max_kv_len %d: at most %d", max_kv, KV_MAX_KEYS);
    if ((int64_t)B * max_kv > KV_MAX_ALL_KEYS)
        return fail(W4A16_ERR_UNSUPPORTED, "%d sequences with max_kv_len %d: at most 2^36 keys in a call", B, max_kv);
    if (B > 65535) return fail(W4A16_ERR_UNSUPPORTED, "%d sequences: at most 65535 in a call", B);
    if (T > KV_MAX_ROWS / Hq) return fail(W4A16_ERR_UNSUPPORTED, "%d queries of %d heads: at most %d in a call", T, Hq, KV_MAX_ROWS);
    const KvAttnShape s = kv_attention_shape(f, T, B, Hq, Hkv, D, max_q, max_kv);
    if (s.many ? (int64_t)s.tiles * s.splits > 65535 : s.places > 65535)
        return fail(W4A16_ERR_UNSUPPORTED, "max_q_len %d with max_kv_len %d: too many tiles for one call", max_q, max_kv);
    return W4A16_OK;
}

size_t kv_attention_workspace_size(const KvFormat& f, int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D,
                                   int32_t max_q_len, int32_t max_kv_len) {
    if (check_attention(f, T, B, Hq, Hkv, D, max_q_len, max_kv_len)) return 0;
    return KV_COUNTER_BYTES + kv_partial_bytes(f, kv_attention_shape(f, T, B, Hq, Hkv, D, max_q_len, max_kv_len), T, B, Hq, Hkv, D, max_kv_len);
}

void kv_path(const KvFormat& f, int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_q_len, int32_t max_kv_len, int32_t* out) {
    const KvAttnShape s = kv_attention_shape(f, T, B, Hq, Hkv, D, max_q_len, max_kv_len);
    const int32_t few[4] = {1, s.nt, s.places, s.join_apart}, many[4] = {2, s.groups, s.splits, s.few_q};
    for (int i = 0; i < 4; ++i) out[i] = s.many ? many[i] : few[i];
}

int kv_attention(const KvFormat& f, void* stream, int elem, const void* q, int32_t q_stride_t, int32_t q_stride_h,
                 const void* cache, const int32_t* page_table, const int32_t* kv_lens, const int32_t* cu_q, void* out,
                 int32_t out_stride_t, int32_t out_stride_h, float* lse, int32_t T, int32_t B, int32_t Hq, int32_t Hkv,
                 int32_t D, int32_t num_pages, int32_t page_size, int32_t pages_per_seq, int32_t max_q_len,
                 int32_t max_kv_len, float scale, int32_t causal, int32_t window, void* workspace, size_t workspace_bytes) {
    if (int rc = check_elem(elem)) return rc;
    if (int rc = check_geometry(num_pages, Hkv, D, page_size)) return rc;
    if (int rc = check_attention(f, T, B, Hq, Hkv, D, max_q_len, max_kv_len)) return rc;
    if (pages_per_seq < 1) return fail(W4A16_ERR_INVALID_ARG, "pages_per_seq (%d) must be positive", pages_per_seq);
    if (window < 0) return fail(W4A16_ERR_INVALID_ARG, "window (%d) must not be negative", window);
    const float scale_log2 = scale * 1.4426950408889634f;
    if (!std::isfinite(scale_log2)) return fail(W4A16_ERR_INVALID_ARG, "scale must be finite, and below 2e38");
    if (!cu_q && T != B) return fail(W4A16_ERR_INVALID_ARG, "without cu_q every sequence has one query (T=%d B=%d)", T, B);
    if (!cu_q && max_q_len != 1) return fail(W4A16_ERR_INVALID_ARG, "without cu_q max_q_len is 1, not %d", max_q_len);
    if (T == 0 || B == 0) return W4A16_OK;
    if (!cache || !page_table || !kv_lens) return fail(W4A16_ERR_INVALID_ARG, "null pointer argument (cache, page_table or kv_lens)");
    if (!aligned(cache, 16)) return fail(W4A16_ERR_INVALID_ARG, "cache must be 16-byte aligned");
    if (!aligned(page_table, 4) || !aligned(kv_lens, 4) || !aligned(cu_q, 4) || !aligned(lse, 4))
        return fail(W4A16_ERR_INVALID_ARG, "page_table, kv_lens, cu_q and lse must be 4-byte aligned");
    if (int rc = check_rows("q", q, q_stride_t, q_stride_h, T, Hq, D, 8, false)) return rc;
    if (int rc = check_rows("out", out, out_stride_t, out_stride_h, T, Hq, D, 8, true)) return rc;
    const KvAttnShape s = kv_attention_shape(f, T, B, Hq, Hkv, D, max_q_len, max_kv_len);
    const size_t need = KV_COUNTER_BYTES + kv_partial_bytes(f, s, T, B, Hq, Hkv, D, max_kv_len);
    if (!workspace || workspace_bytes < need)
        return fail(W4A16_ERR_INVALID_ARG, "workspace too small (%zu < %zu bytes)", workspace ? workspace_bytes : (size_t)0, need);
    if (!aligned(workspace, 256)) return fail(W4A16_ERR_INVALID_ARG, "workspace must be 256-byte aligned");
    KvAttnParams p{};
    p.q = q; p.out = out; p.lse = lse; p.cache = static_cast<const unsigned char*>(cache);
    p.table = page_table; p.kv_lens = kv_lens; p.cu_q = cu_q;
    p.q_st = q_stride_t; p.q_sh = q_stride_h; p.o_st = out_stride_t; p.o_sh = out_stride_h;
    p.num_pages = num_pages; p.pages_per_seq = pages_per_seq; p.T = T; p.B = B; p.Hq = Hq; p.Hkv = Hkv;
    p.page_shift = __builtin_ctz((unsigned)page_size);
    p.max_kv = max_kv_len;
    p.scale_log2 = scale_log2;
    p.scale_mant = std::frexp(scale_log2, &p.scale_exp); p.causal = causal != 0; p.window = window < (1 << 30) ? window : 1 << 30;
    p.counters = static_cast<uint32_t*>(workspace);
    p.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + KV_COUNTER_BYTES);
    p.G = Hq / Hkv;
    p.least_q = 1; p.most_q = INT32_MAX;
    (void)hipGetLastError();
    const bool bf16 = elem == W4A16_BF16;
    hipStream_t st = static_cast<hipStream_t>(stream);
    hipError_t e = hipSuccess;
    if (s.few_q) {
        const KvAttnShape part = kv_few_part(f, s, T, B, Hq, Hkv, D, max_kv_len);
        KvAttnParams few = p;
        kv_params(f, few, part, D, s.few_q, T);
        few.most_q = s.few_q;
        few.partials += s.partial_bytes / sizeof(float);
        e = f.launch_few(bf16, D, few, part, st);
        p.least_q = s.few_q + 1;
    }
    kv_params(f, p, s, D, max_q_len, T);
    if (e == hipSuccess) e = s.many ? f.launch_many(bf16, D, p, s, st) : f.launch_few(bf16, D, p, s, st);
    return e == hipSuccess ? W4A16_OK : hip_fail(e, f.name);
}

}  // namespace w4a16
