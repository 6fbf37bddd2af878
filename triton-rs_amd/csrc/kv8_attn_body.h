// Attention over the 8-bit key/value cache (kv8.h): what its two kernels share.
//
//   w_j = scale q . k_j,  out = sum_j p_j v_j / sum_j p_j,  p_j = exp(w_j - m),  lse = m + ln sum
// in one pass over the keys with a running reference m (no visible key: out = 0, lse = -infinity).
//
// A block's keys are s_k n and its values s_v n with one power of two each, n in e4m3, which fp16 and bf16 hold
// exactly: the matrix cores take n (two conversions of two bytes for four operands) and q as it is, in q's
// type, so the first product has no rounding but that of its fp32 sum. A scale acts on a whole 16 x 16 tile of logits:
// s_k in the factor that softmax's base 2 needs anyway, s_v as its exponent, added to the logit. What is
// exponentiated is log2(p_j s_v): the weight that the second product takes, rounded to fp16 (2^-12 of it; of what the
// matrix cores take the type with the most bits). The sum of p_j is that of a tile's weights times 1 / s_v; where all of a lane's
// weights of a tile are below 2^-100, which fp32 may not hold although p_j counts (s_v far below the others), p_j is exponentiated by itself. The
// reference m follows the largest weight p_j s_v, which is 2^8 when it is set and 2^15 at most: it is raised (with the sums
// scaled down) only where a weight would pass that, so maxima pass between lanes only then, and a block of
// large values and no weight takes no bits from the others. Scales are 2^-60 to 2^120, so a sum of 2^30 p_j
// stays within 2^-113 and 2^105.
//
// A wave holds 16 NT columns (query rows times the G query heads of one key/value head) and walks the
// keys 32 at a time. With S^T = K Q^T a lane has the logits of one column at tokens 4 (lane / 16) + i of
// either block of 16, which is how the second product takes them as its operand, so no logit or weight passes
// between lanes or through LDS. A column's reference follows what the column sees, nothing else.
#pragma once
#include "kv8.h"
#include "kv_attn_body.h"

namespace w4a16 {

constexpr float KV8_MOST = 15.f;   // p_j s_v <= 2^15
constexpr float KV8_ROOM = 7.f;    // a raise leaves the largest at 2^-7 of that
constexpr float KV8_LOW = -100.f;  // log2 of weights whose p_j is exponentiated by itself

// Two e4m3 bytes (the low or the high ones) of a word in the type of an operand, exactly.
template <typename E, bool HIGH>
__device__ __forceinline__ uint32_t from_e4m3(uint32_t w) {
    if constexpr (__is_same(E, half_t)) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, HIGH));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.f, HIGH));
}
// Eight of them: an operand of the 16 x 16 x 32 product
template <typename E>
__device__ __forceinline__ typename vec8<E>::type operand8(uint32_t lo, uint32_t hi) {
    const u32x4 t = {from_e4m3<E, false>(lo), from_e4m3<E, true>(lo), from_e4m3<E, false>(hi), from_e4m3<E, true>(hi)};
    return __builtin_bit_cast(typename vec8<E>::type, t);
}

// Bytes of a word of values whose tokens 4 kb + i are in [lo, hi) of the block.
__device__ __forceinline__ uint32_t token_bytes(int lo, int hi, int kb) {
    const int a = min(max(lo - 4 * kb, 0), 4), b = min(max(hi - 4 * kb, 0), 4);
    const uint32_t from = a == 4 ? 0u : ~0u << (8 * a), to = b == 4 ? ~0u : ~(~0u << (8 * b));
    return from & to;
}

typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));
// What logits and weights take of a block's last 16 bytes. (there: a token of it is seen; else its scales may be anything, and
// a NaN would pass into the sums by way of weights of zero.)
struct Kv8Scale {
    float key;       // scale of its keys, times scale log2(e)
    float value;     // log2 of the scale of its values
    float back;      // 1 / that scale
    uint32_t nan;    // rows that are not finite
    __device__ __forceinline__ static Kv8Scale of(u32x3 tail, float factor, bool there) {
        const uint32_t e = there ? (tail[1] >> 23) & 255u : 127u;
        return {there ? __uint_as_float(tail[0]) * factor : 0.f, (float)((int)e - 127), __uint_as_float((254u - e) << 23), there ? tail[2] : 0u};
    }
};

// A wave's 16 NT columns.
template <typename E, int D, int NT>
struct Kv8Cols {
    typedef typename vec8<E>::type vec_t;
    static constexpr int KW = D / 32;   // operands of a row of keys
    static constexpr int VT = D / 16;   // 16-row tiles of the result
    int c, n;              // first column, columns (0 or less: none)
    int lo[NT], hi[NT];    // keys that this lane's columns see
    int jlo, jhi;          // keys that some column sees, of the chunk
    int all_lo, all_hi;    // keys that every column sees
    vec_t qf[NT][KW];      // dimensions 64 g + 16 (lane / 16) + 8 h + (0..7) in qf[t][2 g + h]
    float m[NT], l[NT];    // reference and sum of p_j = exp2(logit - m)
    float most[NT];        // KV8_MOST, -infinity until a column has seen a key
    float4_t o[NT][VT];    // of column lane % 16, dimensions (4 (lane / 16) + i) D / 16 + x in o[t][x][i]

    __device__ __forceinline__ void load(const KvAttnParams& p, const KvItem& w, int first_col, int lane) {
        c = first_col;
        n = min(16 * NT, w.n * p.G - c);
        const int col = lane & 15, kb = lane >> 4;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = c + 16 * t + col, i = w.n == 1 ? 0 : r / p.G;
            const bool in = 16 * t + col < n;
            hi[t] = in ? w.see_hi(p, i) : 0;
            lo[t] = in ? w.see_lo(p, i) : 0;
            const uint16_t* src = static_cast<const uint16_t*>(p.q) + (size_t)(w.q0 + i) * p.q_st + (size_t)(w.h * p.G + r - i * p.G) * p.q_sh + 16 * kb;
#pragma unroll
            for (int x = 0; x < KW; ++x) {
                u32x4 v = {0, 0, 0, 0};
                if (in) v = *reinterpret_cast<const u32x4*>(src + 64 * (x >> 1) + 8 * (x & 1));
                qf[t][x] = __builtin_bit_cast(vec_t, v);
            }
        }
        const int i0 = w.n == 1 ? 0 : c / p.G, i1 = w.n == 1 ? 0 : (c + max(n, 1) - 1) / p.G;
        jlo = max(w.k0, w.see_lo(p, i0));
        jhi = n > 0 ? min(w.k1, w.see_hi(p, i1)) : 0;
        all_lo = w.see_lo(p, i1);
        all_hi = w.see_hi(p, i0);
    }
    // Infinities of q become NaN: a query that has one is NaN where it sees a key, as infinite logits have no softmax,
    // while all of them -infinity would look like a query that sees none.
    __device__ __forceinline__ void start() {
        constexpr uint32_t inf = __is_same(E, half_t) ? 0x7C00u : 0x7F80u;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int x = 0; x < KW; ++x) {
                u32x4 v = __builtin_bit_cast(u32x4, qf[t][x]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w = v[e], a = w & 0x7FFFu, b = (w >> 16) & 0x7FFFu;
                    v[e] = w | (a < inf ? 0u : 0x7FFFu) | (b < inf ? 0u : 0x7FFF0000u);
                }
                qf[t][x] = __builtin_bit_cast(vec_t, v);
            }
            m[t] = l[t] = 0.f;
            most[t] = -INFINITY;
#pragma unroll
            for (int x = 0; x < VT; ++x) o[t][x] = float4_t{0.f, 0.f, 0.f, 0.f};
        }
    }

    // The lane's tokens j + 4 kb + (0..3, 16..19) that columns t see: those at [from, to) from the first on, not in
    // a block in `bad`.
    struct Seen {
        int from, to, bad;
        __device__ __forceinline__ bool operator()(int s, int i) const { return (16 * s + i >= from) & (16 * s + i < to) & !((bad >> s) & 1); }
    };
    __device__ __forceinline__ Seen seen(int t, int j, int end, int bad, int kb) const {
        int at = j + 4 * kb;
        asm volatile("" : "+v"(at), "+s"(bad));   // (else kept over the loop: every token's distances, in registers)
        return Seen{lo[t] - at, min(hi[t], end) - at, bad};
    }

    // log2(p_j s_v) of 32 tokens from j on for columns t: acc = q . n of the lane's tokens j + 16 s + 4 kb + i. whole: every
    // column sees all 32 and no row is NaN; else tokens from `end` on and those of blocks in `bad` are not seen. Raises m where
    // a weight would pass 2^15. back: what a block's weights count in the sum of p_j, 1 / s_v (or 0 where they are counted here).
    __device__ __forceinline__ void logits(int t, float (&x)[2][4], float (&back)[2], const float4_t (&acc)[2], const Kv8Scale (&s)[2], bool whole,
                                           int j, int end, int bad, int kb) {
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const float off = s[b].value - m[t];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[b][i] = __builtin_fmaf(acc[b][i], s[b].key, off);
        }
        if (!whole) {
            const Seen in = seen(t, j, end, bad, kb);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if ((s[b].nan >> (4 * kb + i)) & 1) x[b][i] = __builtin_nanf("");
                    if (!in(b, i)) x[b][i] = -INFINITY;
                }
            if ((s[0].nan | s[1].nan) >> 16) {   // a value row of NaN makes those columns NaN that see it
                uint32_t hit = 0;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) hit |= in(b, i) ? (s[b].nan >> (16 + 4 * kb + i)) & 1 : 0u;
                const float add = kb_umax(hit) ? __builtin_nanf("") : 0.f;
#pragma unroll
                for (int y = 0; y < VT; ++y) o[t][y] += add;
            }
        }
        const float low = fminf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])), fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, x[b][i]);
#pragma unroll
        for (int b = 0; b < 2; ++b) back[b] = s[b].back;
        if (__any((top > most[t]) | (low < KV8_LOW))) {   // rare after the first steps
            top = kb_max(top);
            const bool up = top > most[t];
            const float by = up ? top - (KV8_MOST - KV8_ROOM) : 0.f;
            // (a column's first keys: nothing summed yet)
            const float fall = most[t] == -INFINITY ? 0.f : half_fall(0.f, by);
            m[t] += by;
            l[t] = l[t] * fall * fall;
#pragma unroll
            for (int y = 0; y < VT; ++y) o[t][y] *= fall * fall;
            most[t] = up ? KV8_MOST : most[t];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[b][i] -= by;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const bool alone = fmaxf(fmaxf(x[b][0], x[b][1]), fmaxf(x[b][2], x[b][3])) < KV8_LOW;
                float p = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) p += __builtin_amdgcn_exp2f(x[b][i] - s[b].value);
                l[t] += alone ? p : 0.f;
                back[b] = alone ? 0.f : back[b];
            }
        }
    }

    // The weights as operand; the sum of p_j.
    __device__ __forceinline__ half8_t weights(int t, const float (&x)[2][4], const float (&back)[2]) {
        half8_t w;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f[i] = __builtin_amdgcn_exp2f(x[b][i]);
                w[4 * b + i] = (half_t)f[i];
            }
            l[t] = __builtin_fmaf((f[0] + f[1]) + (f[2] + f[3]), back[b], l[t]);
        }
        return w;
    }

    // sums over the lanes of a column
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            l[t] = kb_sum(l[t]);
            if (most[t] == -INFINITY && l[t] == 0.f) m[t] = -FLT_MAX;
        }
    }
};

// What of a block's last 16 bytes says something, in every lane: a vector load, which is waited for with the block's others. (A
// scalar load is waited for with all scalar loads, the next step's among them: 48 sequences of kv8_few.hip 63.9 us, 63.5 so.)
__device__ __forceinline__ u32x3 block_tail(const unsigned char* block, int D) {
    return *reinterpret_cast<const u32x3*>(at_bytes(block, 32 * D + vconst(0)));
}

}  // namespace w4a16
