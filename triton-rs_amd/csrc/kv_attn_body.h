// Attention over a paged key/value cache in fewer bits: what does not depend on how the cache holds its rows.
// kv4_attn_body.h and kv8_attn_body.h have the mathematics.
//
// Query row i of sequence b stands at position kv_len - q_len + i and sees key j < kv_len where
// (causal) j <= its position and (window) j > its position - window.
#pragma once
#include <cfloat>

#include "elements.h"
#include "kv_attn.h"
#include "splitk.h"

namespace w4a16 {

// what a column's sum of weighted values is multiplied by, l = sum of its weights, values held times 2^-DOWN
template <int DOWN>
__device__ __forceinline__ float over_sum(float l) { return l == 0.f ? 0.f : (float)(1 << DOWN) / l; }
// Square root of the factor from reference m to mm: references of steps, waves and chunks may lie further apart than
// fp32's exponents reach (value scales do), where a sum of p_j is far from 1 as well. It is multiplied twice.
__device__ __forceinline__ float half_fall(float m, float mm) { return __builtin_amdgcn_exp2f(0.5f * (m - mm)); }

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

// over the four lanes of a column, 16 apart: each swap of rows or halves with itself leaves a lane's own value and
// its partner's in the two results
template <typename F>
__device__ __forceinline__ float kb_all(float v, F f) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float kb_sum(float v) { return kb_all(v, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ uint32_t kb_umax(uint32_t v) {
    return __float_as_uint(kb_all(__uint_as_float(v), [](float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }));
}
__device__ __forceinline__ float kb_max(float v) { return kb_all(v, [](float a, float b) { return fmaxf(a, b); }); }

// over the lanes of a wave: inclusive f-sums (f(0, v) = v)
template <typename F>
__device__ __forceinline__ int wave_scan(int v, F f) {
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));   // one lane up the row, two, four, eight
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));   // the last of a row to the next
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));   // the last of the lower half to the upper
    return v;
}
__device__ __forceinline__ int wave_sums(int v) { return wave_scan(v, [](int a, int b) { return a + b; }); }

__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f; }

// What a workgroup takes of sequence b, key/value head h: columns from c0 on, of keys [k0, k1) of this chunk.
struct KvItem {
    int h, b, q0, n, len, first;   // first row of q, queries, keys, position of query 0
    int c0, cols;                  // first column, columns from there to the sequence's end
    int split, chunks, k0, k1;
    size_t at;                     // number of (tile, b, h)
    size_t slot;                   // of its first chunk's partial results
    __device__ __forceinline__ int see_hi(const KvAttnParams& p, int i) const { return p.causal ? max(0, min(len, first + i + 1)) : len; }
    __device__ __forceinline__ int see_lo(const KvAttnParams& p, int i) const { return p.window ? max(0, first + i - p.window + 1) : 0; }

    // Sequence b and its columns from c0 on; keys [lo, hi) that they see, lo a multiple of STEP.
    template <int WG_COLS, int STEP>
    __device__ __forceinline__ void sequence(const KvAttnParams& p, int b_, int c0_, int& lo, int& hi) {
        b = b_;
        c0 = c0_;
        // (the loads go out together; without cu_q its place is not looked at)
        const int32_t* cu = p.cu_q ? p.cu_q + b : p.kv_lens;
        const int kv = p.kv_lens[b], cu0 = cu[0], cu1 = p.cu_q ? cu[1] : 0;
        q0 = p.cu_q ? min(max(cu0, 0), p.T) : b;
        const int q1 = p.cu_q ? min(max(cu1, 0), p.T) : b + 1;
        n = min(q1 - q0, p.max_q);
        cols = q1 - q0 < p.least_q || q1 - q0 > p.most_q ? 0 : n * p.G - c0;
        const long long cap = (long long)p.pages_per_seq << p.page_shift;
        len = (int)max(0ll, min((long long)min(kv, p.max_kv), cap));
        first = len - (q1 - q0);
        const int i0 = n <= 1 ? 0 : c0 / p.G, i1 = n <= 1 ? 0 : (min(c0 + WG_COLS, n * p.G) - 1) / p.G;
        hi = see_hi(p, i1);
        lo = min(see_lo(p, i0), hi) & ~(STEP - 1);
    }
    // Chunk split_ of chunks_ of `chunk` keys in [lo, hi).
    __device__ __forceinline__ void take(int split_, int chunks_, int chunk, int lo, int hi) {
        split = split_;
        chunks = chunks_;
        k0 = lo + split * chunk;
        k1 = chunks == 1 ? hi : k0 + min(hi - k0, chunk);
    }
};

// Where a workgroup's results go: out and lse, or (more than one chunk) its slot of fp32 partials.
// A value is its fp32 sum times 2^DOWN over the sum of weights.
template <typename E, int D, int DOWN>
struct KvSink {
    const KvAttnParams& p;
    const KvItem& w;
    float *item, *part, *part_ml;
    size_t slot_floats;
    __device__ __forceinline__ KvSink(const KvAttnParams& p_, const KvItem& w_) : p(p_), w(w_) {
        slot_floats = (size_t)p.slot_cols * (D + 2);
        item = p.partials + w.slot * slot_floats;
        part = item + w.split * slot_floats;
        part_ml = part + (size_t)p.slot_cols * D;
    }
    // column r (of the sequence): row of q and head
    __device__ __forceinline__ void place(int r, int& row, int& head) const {
        const int i = w.n == 1 ? 0 : r / p.G;
        row = w.q0 + i;
        head = w.h * p.G + r - i * p.G;
    }
    __device__ __forceinline__ void out(int r, int d, float4_t v, float inv) const {
        int row, head;
        place(r, row, head);
        uint16_t* dst = static_cast<uint16_t*>(p.out) + (size_t)row * p.o_st + (size_t)head * p.o_sh + d;
        *reinterpret_cast<u32x2*>(dst) = u32x2{pack2(E{}, saturate<E>(v[0] * inv), saturate<E>(v[1] * inv)),
                                               pack2(E{}, saturate<E>(v[2] * inv), saturate<E>(v[3] * inv))};
    }
    __device__ __forceinline__ void out8(int r, int d, float4_t v, float4_t u, float inv) const {
        int row, head;
        place(r, row, head);
        uint16_t* dst = static_cast<uint16_t*>(p.out) + (size_t)row * p.o_st + (size_t)head * p.o_sh + d;
        *reinterpret_cast<u32x4*>(dst) = u32x4{pack2(E{}, saturate<E>(v[0] * inv), saturate<E>(v[1] * inv)),
                                               pack2(E{}, saturate<E>(v[2] * inv), saturate<E>(v[3] * inv)),
                                               pack2(E{}, saturate<E>(u[0] * inv), saturate<E>(u[1] * inv)),
                                               pack2(E{}, saturate<E>(u[2] * inv), saturate<E>(u[3] * inv))};
    }
    __device__ __forceinline__ void lse(int r, float m, float l) const {
        if (!p.lse) return;
        int row, head;
        place(r, row, head);
        p.lse[(size_t)row * p.Hq + head] = lse_of(m, l);
    }
    // four values of column r from dimension d on, unnormalised; its reference and sum
    __device__ __forceinline__ void put(int r, int d, float4_t v, float inv) const {
        if (w.chunks > 1) st_partial4<SCOPE_DEVICE>(part + (size_t)(r - w.c0) * D + d, v);
        else out(r, d, v, inv);
    }
    __device__ __forceinline__ void put_ml(int r, float m, float l) const {
        if (w.chunks > 1) {
            st_partial<SCOPE_DEVICE>(part_ml + 2 * (r - w.c0), m);
            st_partial<SCOPE_DEVICE>(part_ml + 2 * (r - w.c0) + 1, l);
        } else {
            lse(r, m, l);
        }
    }
    // Quad e of values (column e / (D / 4)) over chunks share, share + shares, ...; then over the shares, `span` threads
    // apart, through LDS (256 entries each). on: there is such a quad and share. In order of the chunks within a
    // share, then of the shares. For few columns (kv_few.h): partial results by column.
    __device__ __forceinline__ void join_quads(int e, int share, int shares, int span, bool on, float4_t* vals, float (*ml)[2]) const {
        const int c = on ? e / (D / 4) : 0, d = 4 * (e - c * (D / 4)), chunks = w.chunks;
        const float* at = item + (size_t)c * D + d;
        const float* heads = item + (size_t)p.slot_cols * D + 2 * c;
        float m = -FLT_MAX, l = 0.f;
        float4_t v = {0.f, 0.f, 0.f, 0.f};
        if (on)
            for (int s0 = share; s0 < chunks; s0 += 8 * shares) {
                float4_t x[8];
                uint64_t h[8];
#pragma unroll
                for (int y = 0; y < 8; ++y) {
                    const size_t s = min(s0 + shares * y, chunks - 1);
                    h[y] = __hip_atomic_load(reinterpret_cast<const uint64_t*>(heads + s * slot_floats), __ATOMIC_RELAXED, SCOPE_DEVICE);
                    x[y] = ld_partial4<SCOPE_DEVICE>(at + s * slot_floats);
                }
                float mn = m;
#pragma unroll
                for (int y = 0; y < 8; ++y) mn = fmaxf(mn, __uint_as_float((uint32_t)h[y]));
                const float f = half_fall(m, mn);
                v *= f * f;
                l = l * f * f;
#pragma unroll
                for (int y = 0; y < 8; ++y)
                    if (s0 + shares * y < chunks) {
                        const float g = half_fall(__uint_as_float((uint32_t)h[y]), mn);
                        v += x[y] * (g * g);
                        l += __uint_as_float((uint32_t)(h[y] >> 32)) * g * g;
                    }
                m = mn;
            }
        if (shares > 1) {
            vals[threadIdx.x] = v;
            ml[threadIdx.x][0] = m;
            ml[threadIdx.x][1] = l;
            __syncthreads();
            if (on && share == 0) {
                float mm = m;
                for (int x = 1; x < shares; ++x) mm = fmaxf(mm, ml[threadIdx.x + x * span][0]);
                const float f = half_fall(m, mm);
                v *= f * f;
                l = l * f * f;
                for (int x = 1; x < shares; ++x) {
                    const float g = half_fall(ml[threadIdx.x + x * span][0], mm);
                    v += vals[threadIdx.x + x * span] * (g * g);
                    l += ml[threadIdx.x + x * span][1] * g * g;
                }
                m = mm;
            }
        }
        if (on && share == 0) {
            out(w.c0 + c, d, v, over_sum<DOWN>(l));
            if (d == 0) lse(w.c0 + c, m, l);
        }
    }
    // The last of the chunks to arrive (splitk.h) joins them: 256 threads, `live` columns.
    __device__ __forceinline__ void join(int live, float4_t* vals, float (*ml)[2], int* last) const {
        if (!splitk_arrive(p.counters + w.at, w.chunks, last)) return;
        const int quads = live * (D / 4), shares = quads >= 256 ? 1 : min(256 / quads, 8), span = shares == 1 ? 256 : quads;
        const int share = threadIdx.x / span;
        for (int e0 = 0; e0 < quads; e0 += span) {
            const int e = e0 + threadIdx.x - share * span;
            join_quads(e, share, shares, span, e < quads && share < shares, vals, ml);
        }
    }
    // For many columns, 128 of them with partial results as lanes have them: per column (m, 1 / l) over all
    // chunks, then the values of part `part` of PARTS, two chunks in flight. place(e, c, d): column and dimension of quad e.
    template <int PARTS, typename P>
    __device__ __forceinline__ void join_lanes(int live, float* ml, int part, P place) const {
        const int chunks = w.chunks;
        const float* heads = item + (size_t)p.slot_cols * D;
        if ((int)threadIdx.x < live) {
            float mm = -FLT_MAX, ll = 0.f;
            for (int s = 0; s < chunks; ++s) {
                const uint64_t x = __hip_atomic_load(reinterpret_cast<const uint64_t*>(heads + s * slot_floats + 2 * threadIdx.x), __ATOMIC_RELAXED, SCOPE_DEVICE);
                const float mx = __uint_as_float((uint32_t)x), mn = fmaxf(mm, mx);
                const float f = half_fall(mm, mn), g = half_fall(mx, mn);
                ll = ll * f * f + __uint_as_float((uint32_t)(x >> 32)) * g * g;
                mm = mn;
            }
            ml[2 * threadIdx.x] = mm;
            ml[2 * threadIdx.x + 1] = over_sum<DOWN>(ll);
            if (part == 0) lse(w.c0 + threadIdx.x, mm, ll);
        }
        __syncthreads();
        constexpr int QUADS = 32 * D / PARTS;   // of 128 columns
        static_assert(QUADS % 256 == 0, "whole rounds");
#pragma unroll 1
        for (int e = part * QUADS + threadIdx.x; e < (part + 1) * QUADS; e += 256) {
            int c, d;
            place(e, c, d);
            const int at = min(c, live - 1);
            const float mm = ml[2 * at];
            float4_t v = {0.f, 0.f, 0.f, 0.f};
            for (int s0 = 0; s0 < chunks; s0 += 2) {
                float4_t x[2];
                float f[2];
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const size_t s = min(s0 + y, chunks - 1);
                    f[y] = __hip_atomic_load(heads + s * slot_floats + 2 * at, __ATOMIC_RELAXED, SCOPE_DEVICE);
                    x[y] = ld_partial4<SCOPE_DEVICE>(item + s * slot_floats + 4 * e);
                }
#pragma unroll
                for (int y = 0; y < 2; ++y)
                    if (s0 + y < chunks) v += x[y] * __builtin_amdgcn_exp2f(f[y] - mm);
            }
            if (c < live) out(w.c0 + c, d, v, ml[2 * c + 1]);
        }
    }
    // Partial results as lanes have them: number of a quad, and place of quad e
    static constexpr int VT = D / 16;
    __device__ __forceinline__ static int lane_quad(int wave, int t, int i, int x, int lane) {
        return (((wave * 2 + t) * 4 + i) * (VT / 4) + x / 4) * 64 + lane;
    }
    __device__ __forceinline__ static void lane_place(int e, int& c, int& d) {
        const int lane = e & 63, q = e >> 6, x = q % (VT / 4), r = q / (VT / 4);
        c = 16 * (r >> 2) + (lane & 15);
        d = (4 * (lane >> 4) + (r & 3)) * VT + 4 * x;
    }
};

// Pages of a sequence, clamped to its keys (len > 0).
struct KvPages {
    const int32_t* table;
    const unsigned char* heads;   // head h of page 0
    size_t page_bytes;
    int bshift, last, num_pages, block_bytes;
    __device__ __forceinline__ KvPages(const KvAttnParams& p, const KvItem& w, int block) {
        table = p.table + (size_t)w.b * p.pages_per_seq;
        bshift = p.page_shift - 4;
        last = (w.len - 1) >> 4;
        num_pages = p.num_pages;
        block_bytes = block;
        page_bytes = ((size_t)p.Hkv * block) << bshift;
        heads = p.cache + (((size_t)w.h * block) << bshift);
    }
    // (constant address space: a scalar load, also behind LDS loads written in asm, that is not counted with them)
    __device__ __forceinline__ int page(int blk) const {
        return ((const __attribute__((address_space(4))) int32_t*)table)[min(blk, last) >> bshift];
    }
    __device__ __forceinline__ bool ok(int page) const { return (unsigned)page < (unsigned)num_pages; }
    __device__ __forceinline__ const unsigned char* block(int page, int blk) const {
        return heads + (ok(page) ? (size_t)page * page_bytes : 0) + (size_t)(min(blk, last) & ((1 << bshift) - 1)) * block_bytes;
    }
};

}  // namespace w4a16
