// Attention over the 4-bit key/value cache (kv4.h): what its two kernels share.
//
// Query row i of sequence b stands at position kv_len - q_len + i and sees key j < kv_len where
// (causal) j <= its position and (window) j > its position - window:
//   w_j = scale q . k_j,  out = sum_j p_j v_j / sum_j p_j,  p_j = exp(w_j - m),  lse = m + ln sum
// in one pass over the keys with a running reference m (no visible key: out = 0, lse = -infinity).
//
// A row of keys is s (n - z), so q . k = s (q . (n - z)), and sum_j p_j v_j is sum_j (p_j s_j) (n_j - z_j):
// the matrix cores (v_mfma_f32_16x16x32_f16) take the integers n - z and a scale acts on one logit or
// weight a token. Masked out of its word into 0x6400 a nibble is the fp16 number 1024 + n (1024 + 16 n
// from bits 4..7 of a half); one packed subtraction of 1024 + z, or fma with 1/16 and 64 + z, gives
// n - z exactly: nine instructions for eight operands. (A nibble left as the fp16 subnormal that it is
// without the 0x6400 needs five, but the matrix cores align a sum's terms by the exponents that their
// operands show, and a subnormal shows 2^-14: errors of 2^-12 of the largest term.)
//
// A wave holds 16 NT columns (query rows times the G query heads of one key/value head) and walks the
// keys 32 at a time. With S^T = K Q^T a lane has the logits of one column at tokens 4 (lane / 16) + i of
// either block of 16, which is how the second product takes them as its operand (the sum over the
// tokens may run in any order as long as the values follow), so no logit or weight passes between lanes
// or through LDS. q is scaled by powers of two into fp16's range: exactly for fp16, for bf16 but for what
// lies 2^24 below a row's largest. A weight p_j s_j is rounded to fp16 (2^-11, of what the matrix
// cores take the type with the most bits); the reference m is such that the largest of them is 2^7 when it is set and
// 2^15 at most, so it follows logits and value scales together: a row of large values and no weight takes no bits
// from the others. It is raised (with the sums scaled down) only where a step's largest logit and largest value
// scale would pass 2^15, so maxima pass between lanes only then. A column's reference follows what the column sees,
// nothing else. Sums are fp32.
#pragma once
#include <cfloat>

#include "device_common.h"
#include "kv4.h"
#include "splitk.h"

namespace w4a16 {

constexpr float KV4_MOST = 15.f;   // p_j s_j <= 2^15
constexpr float KV4_ROOM = 7.f;    // a raise leaves the largest at 2^-7 to 2^-8 of that
// Value scales are taken times 2^-VALUE_DOWN, and smaller ones than LEAST_SCALE (all zero in fp16) as that in the
// reference: p_j stays between 2^-98, at the largest bf16 scale, and 2^95, so that a sum of 2^30 fits fp32.
template <typename E>
constexpr int VALUE_DOWN = __is_same(E, half_t) ? 0 : 20;
template <typename E>
constexpr float LEAST_SCALE = __is_same(E, half_t) ? 0x1p-24f : 0x1p-80f;

template <typename E>
__device__ __forceinline__ float param_scale(uint32_t w) {
    if constexpr (__is_same(E, half_t)) return (float)__builtin_bit_cast(half_t, (uint16_t)w);
    else return bf16_bits_to_f32(w);   // the shift drops the upper half
}

template <typename E>
__device__ __forceinline__ float value_scale(uint32_t w) {
    if constexpr (VALUE_DOWN<E> == 0) return param_scale<E>(w);
    else return param_scale<E>(w) * (1.f / (1 << VALUE_DOWN<E>));
}
// log2 of a number above value scales, from the bits of their largest (NaN beyond all numbers), of `least` at least
__device__ __forceinline__ float log2_above(uint32_t top, uint32_t least) { return (float)((int)(max(top, least) >> 23) - 126); }
constexpr uint32_t INF_BITS32 = 0x7F800000u;
// what sum_j (p_j s_j) (n_j - z_j) is multiplied by, l = sum_j p_j
template <typename E>
__device__ __forceinline__ float over_sum(float l) { return l == 0.f ? 0.f : (float)(1 << VALUE_DOWN<E>) / l; }
// Square root of the factor from reference m to mm: references of steps, waves and chunks may lie further apart than
// fp32's exponents reach (value scales do), where a sum of p_j is far from 1 as well. It is multiplied twice.
__device__ __forceinline__ float half_fall(float m, float mm) { return __builtin_amdgcn_exp2f(0.5f * (m - mm)); }

__device__ __forceinline__ half8_t as_h8(half2_t a, half2_t b, half2_t c, half2_t d) {
    const u32x4 t = {as_u32(a), as_u32(b), as_u32(c), as_u32(d)};
    return __builtin_bit_cast(half8_t, t);
}

// n - z of the nibbles at bits 0 and 16 of x, z1 = 1024 + z; of those at bits 4 and 20, z16 = 64 + z
__device__ __forceinline__ half2_t centred(uint32_t x, half2_t z1) { return nib_pair(x) - z1; }
__device__ __forceinline__ half2_t centred16(uint32_t x, half2_t z16) {
    return __builtin_elementwise_fma(nib_pair16(x), half2_t{(half_t)0.0625f, (half_t)0.0625f}, -z16);
}
// a pair of zero points (one in each half) as 1024 + z and 64 + z
__device__ __forceinline__ half2_t zero1024(uint32_t z) { return as_h2(z | 0x64006400u); }
__device__ __forceinline__ half2_t zero64(uint32_t z) { return as_h2((z << 4) | 0x54005400u); }
// zero points out of parameter words: of one, twice; of two
__device__ __forceinline__ uint32_t zeros_of(uint32_t w) { return perm(0u, w, 0x03020302u); }
__device__ __forceinline__ uint32_t zeros_of(uint32_t lo, uint32_t hi) { return perm(hi, lo, 0x07060302u); }

// the operand of a word of keys: dimensions 8 w + (0, 4, 1, 5, 2, 6, 3, 7) of the lane's quarter row
__device__ __forceinline__ half8_t key_operand(uint32_t x, half2_t z1, half2_t z16) {
    const uint32_t y = x >> 8;
    return as_h8(centred(x, z1), centred16(x, z16), centred(y, z1), centred16(y, z16));
}
// a pair of tokens' values at nibble e (0..3) of their halves of x
template <int EI>
__device__ __forceinline__ half2_t value_pair(uint32_t x, half2_t z1, half2_t z16) {
    const uint32_t y = EI & 2 ? x >> 8 : x;
    return EI & 1 ? centred16(y, z16) : centred(y, z1);
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

template <typename E>
__device__ __forceinline__ float saturate(float v) {
    constexpr float most = __is_same(E, half_t) ? 65504.f : 0x1.fep127f;
    return v > most ? most : v < -most ? -most : v;   // (NaN stays)
}

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
struct Kv4Item {
    int h, b, q0, n, len, first;   // first row of q, queries, keys, position of query 0
    int c0, cols;                  // first column, columns from there to the sequence's end
    int split, chunks, k0, k1;
    size_t at;                     // number of (tile, b, h)
    size_t slot;                   // of its first chunk's partial results
    __device__ __forceinline__ int see_hi(const Kv4AttnParams& p, int i) const { return p.causal ? max(0, min(len, first + i + 1)) : len; }
    __device__ __forceinline__ int see_lo(const Kv4AttnParams& p, int i) const { return p.window ? max(0, first + i - p.window + 1) : 0; }

    // Sequence b and its columns from c0 on; keys [lo, hi) that they see, lo a multiple of STEP.
    template <int WG_COLS, int STEP>
    __device__ __forceinline__ void sequence(const Kv4AttnParams& p, int b_, int c0_, int& lo, int& hi) {
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

// A wave's 16 NT columns.
template <typename E, int D, int NT>
struct Kv4Cols {
    static constexpr int KW = D / 32;   // words of a lane's quarter row of keys: MFMAs of a block
    static constexpr int VT = D / 16;   // 16-row tiles of the result
    int c, n;              // first column, columns (0 or less: none)
    int lo[NT], hi[NT];    // keys that this lane's columns see
    int jlo, jhi;          // keys that some column sees, of the chunk
    int all_lo, all_hi;    // keys that every column sees
    half8_t qf[NT][KW];
    float kscale;          // logits in base 2 are 2^shift kscale s (q . (n - z)), shift 0 but for numbers far from 1
    int shift[NT];         // (of column lane % 16) or from the others'
    uint32_t least;        // for log2_above: LEAST_SCALE, or (some shift is not 0) infinity: every step goes to uncommon()
    float m[NT], l[NT];    // reference and sum of p_j = exp2(logit - m)
    float most[NT];        // KV4_MOST, -infinity until a column has seen a key
    float4_t o[NT][VT];    // of column lane % 16, dimensions (4 (lane / 16) + i) D / 16 + x in o[t][x][i]

    // the rows of q, as they are
    __device__ __forceinline__ void load(const Kv4AttnParams& p, const Kv4Item& w, int first_col, int lane) {
        c = first_col;
        n = min(16 * NT, w.n * p.G - c);
        const int col = lane & 15, kb = lane >> 4;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = c + 16 * t + col, i = w.n == 1 ? 0 : r / p.G;
            const bool in = 16 * t + col < n;
            hi[t] = in ? w.see_hi(p, i) : 0;
            lo[t] = in ? w.see_lo(p, i) : 0;
            const uint16_t* src = static_cast<const uint16_t*>(p.q) + (size_t)(w.q0 + i) * p.q_st + (size_t)(w.h * p.G + r - i * p.G) * p.q_sh + kb * (D / 4);
#pragma unroll
            for (int x = 0; x < KW; ++x) {
                u32x4 v = {0, 0, 0, 0};
                if (in) v = *reinterpret_cast<const u32x4*>(src + 8 * x);
                qf[t][x] = __builtin_bit_cast(half8_t, v);
            }
        }
        const int i0 = w.n == 1 ? 0 : c / p.G, i1 = w.n == 1 ? 0 : (c + max(n, 1) - 1) / p.G;
        jlo = max(w.k0, w.see_lo(p, i0));
        jhi = n > 0 ? min(w.k1, w.see_hi(p, i1)) : 0;
        all_lo = w.see_lo(p, i1);
        all_hi = w.see_hi(p, i0);
    }

    // |q| of the wave's rows, infinities and NaN aside: the largest of each column, the largest and the smallest of these
    // (zeros aside). Infinities become NaN: a query that has one is NaN where it sees a key, as infinite logits have no
    // softmax, while all of them -infinity would look like a query that sees none.
    struct Sizes { float top, low, own[NT]; };
    __device__ __forceinline__ Sizes sizes() {
        typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
        constexpr uint32_t inf = __is_same(E, half_t) ? 0x7C00u : 0x7F80u;
        uint32_t most[NT], low = ~0u, top = 0;   // (bits of non-negative numbers are ordered)
        bool odd = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            ushort2_t m = {0, 0};
#pragma unroll
            for (int x = 0; x < KW; ++x) {
                const u32x4 v = __builtin_bit_cast(u32x4, qf[t][x]);
#pragma unroll
                for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(ushort2_t, v[e] & 0x7FFF7FFFu));
            }
            most[t] = max((uint32_t)m[0], (uint32_t)m[1]);
            odd |= most[t] >= inf;
        }
        if (__any(odd)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                most[t] = 0;
#pragma unroll
                for (int x = 0; x < KW; ++x) {
                    u32x4 v = __builtin_bit_cast(u32x4, qf[t][x]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t a = (v[e >> 1] >> (16 * (e & 1))) & 0x7FFFu;
                        most[t] = max(most[t], a < inf ? a : 0u);
                        v[e >> 1] |= a < inf ? 0u : 0x7FFFu << (16 * (e & 1));
                    }
                    qf[t][x] = __builtin_bit_cast(half8_t, v);
                }
            }
        }
        Sizes r;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            most[t] = kb_umax(most[t]);
            r.own[t] = param_scale<E>(most[t]);
            top = max(top, most[t]);
            low = min(low, most[t] - 1);   // (0 as the largest)
        }
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) {
            top = max(top, (uint32_t)__shfl_xor((int)top, x));
            low = min(low, (uint32_t)__shfl_xor((int)low, x));
        }
        r.top = param_scale<E>(top);
        r.low = param_scale<E>(low == ~0u ? top : low + 1);
        return r;
    }
    // The power of two that takes queries of which `top` is the largest into fp16: to 2^13 to 2^14, or (fp16, whose own
    // range is enough: no bit is lost upwards) less where they are small, more where they are larger.
    __device__ __forceinline__ static int power(float top) {
        constexpr bool F16 = __is_same(E, half_t);
        return top > 0.f ? min(F16 ? 15 : 126, max(F16 ? 0 : -114, 13 - exponent(top))) : 0;
    }
    __device__ __forceinline__ static int exponent(float v) { return (int)(__float_as_uint(v) >> 23) - 127; }

    // q in operand order under the power of two of the largest of the rows; bf16 rows whose own largest is less than 2^-6
    // of it have one of their own, so that what lies 2^24 below a row's largest loses bits at most. (r.top, r.low: of the
    // wave's rows or more, the same in all waves that share kscale and least.)
    __device__ __forceinline__ void start(const Kv4AttnParams& p, const Sizes& r) {
        constexpr bool F16 = __is_same(E, half_t);
        constexpr int APART = 6;
        const int e2 = power(r.top), far = exponent(r.top) - APART;
        // a key scale (below 2^126) times kscale does not overflow, and what is below fp32's normal range is of no
        // account in a logit; the rest of the factor comes last
        const int e = __builtin_amdgcn_readfirstlane(p.scale_exp - e2), a = min(-1, max(-60, e));
        kscale = p.scale_mant * pow2(a);
        least = __any(e != a || (!F16 && exponent(r.low) < far)) ? INF_BITS32 : __builtin_bit_cast(uint32_t, LEAST_SCALE<E>);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int et = !F16 && r.own[t] > 0.f && exponent(r.own[t]) < far ? power(r.own[t]) : e2;
            const float up = pow2(et);
            shift[t] = p.scale_exp - et - a;
#pragma unroll
            for (int x = 0; x < KW; ++x) {
                const u32x4 v = __builtin_bit_cast(u32x4, qf[t][x]);
                half2_t a[4];   // dimensions (0, 1), (2, 3), (4, 5), (6, 7)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (F16) a[e] = as_h2(v[e]) * half2_t{(half_t)up, (half_t)up};
                    else a[e] = half2_t{(half_t)(param_scale<E>(v[e]) * up), (half_t)(param_scale<E>(v[e] >> 16) * up)};
                }
                // dimension e meets the nibble at bits 4 e: operand slot 2 (e % 4) + e / 4
                const uint32_t w01 = as_u32(a[0]), w23 = as_u32(a[1]), w45 = as_u32(a[2]), w67 = as_u32(a[3]);
                qf[t][x] = as_h8(as_h2(perm(w45, w01, 0x05040100u)), as_h2(perm(w45, w01, 0x07060302u)),
                                 as_h2(perm(w67, w23, 0x05040100u)), as_h2(perm(w67, w23, 0x07060302u)));
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

    // What few steps need before their logits: those with a value scale of NaN, or all where a `shift` is not 0. (Two tests, and
    // two branches of either column tile, cost 1024 queries over 32768 keys 690 us, 683 two tests in one place.)
    __device__ __forceinline__ void uncommon(float4_t (&acc)[NT][2], float (&ks)[2][4], float (&vs)[2][4], float above, bool whole, int j,
                                             int end, int bad, int kb) {
        if (__builtin_expect(!__any(above > 128.f), 1)) return;
        if (least == INF_BITS32) {   // the whole factor, on the products
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[t][s][i] = __builtin_ldexpf(acc[t][s][i] * ks[s][i], shift[t]);
                    ks[s][i] = 1.f;
                }
        }
        if (!whole) value_nan(vs, j, end, bad, kb);
    }
    // A value row of NaN (its scale is) makes those columns NaN that see it, whatever its weight, and no others. Where all
    // see it its weights do that; here, where some do not, they become 0 and the columns NaN by themselves.
    __device__ __forceinline__ void value_nan(float (&vs)[2][4], int j, int end, int bad, int kb) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const Seen in = seen(t, j, end, bad, kb);
            uint32_t hit = 0;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) hit |= (in(s, i) & (vs[s][i] != vs[s][i])) ? 1u : 0u;
            const float add = kb_umax(hit) ? __builtin_nanf("") : 0.f;
#pragma unroll
            for (int x = 0; x < VT; ++x) o[t][x] += add;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) vs[s][i] = fmaxf(vs[s][i], 0.f);
    }

    // Logits less m of 32 tokens from j on for columns t: acc = q . (n - z), ks = key scale times kscale, of the
    // lane's tokens j + 16 s + 4 kb + i; vs = value scales, 2^above more than any of them. whole: every column sees
    // all 32; else tokens from `end` on and those of blocks in `bad` are not seen. Raises m where a weight may pass 2^15.
    __device__ __forceinline__ void logits(int t, float (&x)[2][4], const float4_t (&acc)[2], const float (&ks)[2][4], const float (&vs)[2][4],
                                           float above, bool whole, int j, int end, int bad, int kb) {
        float top = -INFINITY;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[s][i] = __builtin_fmaf(acc[s][i], ks[s][i], -m[t]);
        if (!whole) {
            const Seen in = seen(t, j, end, bad, kb);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!in(s, i)) x[s][i] = -INFINITY;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, x[s][i]);
        if (__any(top > most[t] - above)) {   // rare after the first steps
            top = -INFINITY;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = vs[s][i];
                    asm volatile("" : "+v"(v));   // (else all steps take the scales' exponents ahead: 740 us for the 668 of kv4_many.hip)
                    top = fmaxf(top, x[s][i] + log2_above(__float_as_uint(fmaxf(v, LEAST_SCALE<E>)), 0u));   // (NaN as the least)
                }
            top = kb_max(top);
            const bool up = top > most[t];
            const float by = up ? top - (KV4_MOST - KV4_ROOM) : 0.f;
            // (a column's first keys: nothing summed yet)
            const float fall = most[t] == -INFINITY ? 0.f : half_fall(0.f, by);
            m[t] += by;
            l[t] = l[t] * fall * fall;
#pragma unroll
            for (int y = 0; y < VT; ++y) o[t][y] *= fall * fall;
            most[t] = up ? KV4_MOST : most[t];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[s][i] -= by;
        }
    }

    // Their weights p_j s_j as operand; the sum of p_j.
    __device__ __forceinline__ half8_t weights(int t, const float (&x)[2][4], const float (&vs)[2][4]) {
        half8_t w;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float pj = __builtin_amdgcn_exp2f(x[s][i]);
                l[t] += pj;
                w[4 * s + i] = (half_t)(pj * vs[s][i]);
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

// Where a workgroup's results go: out and lse, or (more than one chunk) its slot of fp32 partials.
template <typename E, int D>
struct Kv4Sink {
    const Kv4AttnParams& p;
    const Kv4Item& w;
    float *item, *part, *part_ml;
    size_t slot_floats;
    __device__ __forceinline__ Kv4Sink(const Kv4AttnParams& p_, const Kv4Item& w_) : p(p_), w(w_) {
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
    // share, then of the shares. For kv4_few.hip: partial results by column.
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
            out(w.c0 + c, d, v, over_sum<E>(l));
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
    // For kv4_many.hip, 128 columns of partial results as lanes have them: per column (m, 1 / l) over all
    // chunks, then the values of part `part` of PARTS, two chunks in flight.
    template <int PARTS>
    __device__ __forceinline__ void join_lanes(int live, float* ml, int part) const {
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
            ml[2 * threadIdx.x + 1] = over_sum<E>(ll);
            if (part == 0) lse(w.c0 + threadIdx.x, mm, ll);
        }
        __syncthreads();
        constexpr int QUADS = 32 * D / PARTS;   // of 128 columns
        static_assert(QUADS % 256 == 0, "whole rounds");
#pragma unroll 1
        for (int e = part * QUADS + threadIdx.x; e < (part + 1) * QUADS; e += 256) {
            int c, d;
            lane_place(e, c, d);
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
struct Kv4Pages {
    const int32_t* table;
    const unsigned char* heads;   // head h of page 0
    size_t page_bytes;
    int bshift, last, num_pages, block_bytes;
    __device__ __forceinline__ Kv4Pages(const Kv4AttnParams& p, const Kv4Item& w, int block) {
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
