// Attention over the 4-bit key/value cache (kv4.h).
//
// Query row i of sequence b stands at position kv_len - q_len + i and sees key j < kv_len where
// (causal) j <= its position and (window) j > its position - window:
//   w_j = scale q . k_j,  out = sum_j p_j v_j / sum_j p_j,  p_j = exp(w_j - m),  lse = m + ln sum
// in one pass over the keys with a running reference m (no visible key: out = 0, lse = -infinity).
//
// A row of keys is s (n - z), so q . k = s (q . (n - z)), and sum_j p_j v_j is sum_j (p_j s_j) (n_j - z_j):
// the matrix cores (v_mfma_f32_16x16x32_f16) take the integers n - z and a scale acts on one logit or
// weight a token. Masked out of its word into 0x6400 (0x64006400 for two) a nibble is the fp16 number
// 1024 + n (1024 + 16 n from bits 4..7 of a half); one packed subtraction of 1024 + z, or fma with 1/16
// and 64 + z, gives n - z exactly: nine instructions for eight operands. (A nibble left as the fp16
// subnormal that it is without the 0x6400 needs five, but the matrix cores align a sum's terms by the
// exponents that their operands show, and a subnormal shows 2^-14: errors of 2^-12 of the largest term.)
//
// A wave holds 16 NT columns (query rows times the G query heads of one key/value head) and walks the
// keys 32 at a time. With S^T = K Q^T a lane has the logits of one column at tokens 4 (lane / 16) + i of
// either block of 16, which is how the second product takes them as its operand (the sum over the
// tokens may run in any order as long as the values follow), so nothing passes between lanes or
// through LDS until the end. q is scaled by a power of two (wave-wide) into fp16's range, exactly for fp16
// and bf16 alike. The weights p_j s_j are rounded to fp16 under a wave-wide power of two of the largest
// s_j; m is raised only where a logit passes it by 8 (in base 2), so a tile's maxima pass between lanes
// only then.
//
// A workgroup of four waves takes up to 64 NT columns; where there are fewer (decode), its waves share
// the columns and split the keys, and join through LDS. Long sequences are split over workgroups in
// chunks; the last one to arrive joins their fp32 partials in order (splitk.h's protocol).
#include <algorithm>
#include <cfloat>

#include "device_common.h"
#include "kv4.h"
#include "splitk.h"

namespace w4a16 {

constexpr int KV4_TILE = 32;              // keys of one step
constexpr float RAISE = 8.0f;             // p_j <= 2^8
constexpr int WEIGHT_LOG2 = 7;            // weights, p_j s_j 2^7 / sref, are below 2^14

template <typename E>
__device__ __forceinline__ float param_scale(uint32_t w) {
    if constexpr (__is_same(E, half_t)) return (float)__builtin_bit_cast(half_t, (uint16_t)w);
    else return bf16_bits_to_f32(w);   // the shift drops the upper half
}

// One step's data of a lane: keys of token lane % 16 (a quarter row), values of tokens 4 (lane / 16)..+3
// (a column), the parameters of those four tokens; of two blocks.
template <int D>
struct KvTile {
    uint32_t k[2][D / 32], v[2][D / 32];
    uint32_t kc[2];      // the parameters of the keys' token lane % 16
    u32x4 kp[2], vp[2];
};

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&dst)[N], const unsigned char* base, uint32_t off) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const u32x4 t = *reinterpret_cast<const u32x4*>(at_bytes(base, off + 16 * i));
#pragma unroll
            for (int e = 0; e < 4; ++e) dst[4 * i + e] = t[e];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const u32x2 t = *reinterpret_cast<const u32x2*>(at_bytes(base, off + 8 * i));
            dst[2 * i] = t[0];
            dst[2 * i + 1] = t[1];
        }
    }
}

template <int D>
__device__ __forceinline__ void load_tile(KvTile<D>& t, const unsigned char* b0, const unsigned char* b1, int lane) {
    const uint32_t ko = (lane & 15) * (D / 2) + (lane >> 4) * (D / 8), vo = 8 * D + lane * (D / 8), po = 16 * D + (lane >> 4) * 16;
    load_words(t.k[0], b0, ko);
    load_words(t.k[1], b1, ko);
    t.kc[0] = *reinterpret_cast<const uint32_t*>(at_bytes(b0, 16 * D + (lane & 15) * 4));
    t.kc[1] = *reinterpret_cast<const uint32_t*>(at_bytes(b1, 16 * D + (lane & 15) * 4));
    t.kp[0] = *reinterpret_cast<const u32x4*>(at_bytes(b0, po));
    t.kp[1] = *reinterpret_cast<const u32x4*>(at_bytes(b1, po));
    load_words(t.v[0], b0, vo);
    load_words(t.v[1], b1, vo);
    t.vp[0] = *reinterpret_cast<const u32x4*>(at_bytes(b0, po + 64));
    t.vp[1] = *reinterpret_cast<const u32x4*>(at_bytes(b1, po + 64));
}

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

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

template <typename E>
__device__ __forceinline__ float saturate(float v) {
    constexpr float most = __is_same(E, half_t) ? 65504.f : 0x1.fep127f;
    return v > most ? most : v < -most ? -most : v;   // (NaN stays)
}

__device__ __forceinline__ float kb_sum(float v) {   // over the four lanes of a column
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float kb_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f; }

template <typename E, int D, int NT>
__global__ __launch_bounds__(256, NT == 1 && D <= 128 ? 3 : 2) void kv4_attention_kernel(Kv4AttnParams p) {
    constexpr int KW = D / 32;         // words of a lane's quarter row, MFMAs of a block of keys
    constexpr int VT = D / 16;         // 16-row tiles of the result
    constexpr int COLS = 16 * NT;      // columns of a wave
    constexpr int ROW = D + 4;         // LDS row of a column's result
    __shared__ float red[4][16 * ROW];
    __shared__ float ml[4][COLS][2];
    __shared__ int last;

    const int h = blockIdx.x, b = blockIdx.y;
    const int split = p.splits == 1 ? 0 : blockIdx.z % p.splits;
    const int tile = p.tiles - 1 - (p.splits == 1 ? blockIdx.z : blockIdx.z / p.splits);   // the longest first
    const int q0 = p.cu_q ? min(max(p.cu_q[b], 0), p.T) : b;
    const int q1 = p.cu_q ? min(max(p.cu_q[b + 1], 0), p.T) : b + 1;
    const int n = min(q1 - q0, p.max_q), G = p.G;
    const int c0 = tile * (4 * COLS);
    const int cols = n * G - c0;       // columns from this workgroup's first on
    if (cols <= 0) return;
    const long long cap = (long long)p.pages_per_seq << p.page_shift;
    const int len = (int)max(0ll, min((long long)min(p.kv_lens[b], p.max_kv), cap));
    const int first = len - (q1 - q0);   // position of query 0

    // waves: `groups` groups of columns, each of kspl waves that take every kspl-th step of the keys
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kshift = cols <= COLS ? 2 : cols <= 2 * COLS ? 1 : 0, kspl = 1 << kshift;
    const int cw = c0 + (wave >> kshift) * COLS;   // this wave's first column
    const int col = lane & 15, kb = lane >> 4;

    // keys that some column of the workgroup sees, and this workgroup's chunk of them
    const int i0 = c0 / G, i1 = (min(c0 + 4 * COLS, n * G) - 1) / G;
    const int see_hi = p.causal ? max(0, min(len, first + i1 + 1)) : len;
    const int see_lo = (p.window ? min(max(0, first + i0 - p.window + 1), see_hi) : 0) & ~(KV4_TILE - 1);
    const int chunk = kspl == 1 ? p.chunk_full : p.chunk_thin;
    const int chunks = p.splits == 1 ? 1 : max(1, (int)(((unsigned)(see_hi - see_lo) + chunk - 1) / (unsigned)chunk));
    if (split >= chunks) return;
    const int k0 = p.splits == 1 ? see_lo : see_lo + split * chunk;
    const int k1 = p.splits == 1 ? see_hi : min(see_hi, k0 + chunk);

    // this wave's columns: query rows, what they see, q in operand order
    const int ncol = min(COLS, n * G - cw);   // <= 0: none
    int lo[NT], hi[NT], row[NT], head[NT];
    half8_t qf[NT][KW];
    float qmax = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = cw + 16 * t + col, i = r / G;
        const bool in = 16 * t + col < ncol;
        row[t] = in ? q0 + i : -1;
        head[t] = h * G + (r - i * G);
        hi[t] = !in ? 0 : p.causal ? min(len, first + i + 1) : len;
        lo[t] = in && p.window ? first + i - p.window + 1 : 0;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
            u32x4 x = {0, 0, 0, 0};
            if (in) x = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p.q) + (size_t)row[t] * p.q_st + (size_t)head[t] * p.q_sh + kb * (D / 4) + 8 * w);
            qf[t][w] = __builtin_bit_cast(half8_t, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float a = fabsf(param_scale<E>(x[e])), c = fabsf(param_scale<E>(x[e] >> 16));
                qmax = fmaxf(qmax, a < INFINITY ? a : 0.f);
                qmax = fmaxf(qmax, c < INFINITY ? c : 0.f);
            }
        }
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) qmax = fmaxf(qmax, __shfl_xor(qmax, x));
    // q 2^qe has its largest value in [2^13, 2^14) (or all of it is zero); sums over D nibble products stay finite
    const int qe = qmax > 0.f ? min(100, max(-100, 13 - (int)(__float_as_uint(qmax) >> 23) + 127)) : 0;
    const float qup = pow2(qe);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int w = 0; w < KW; ++w) {
            const u32x4 x = __builtin_bit_cast(u32x4, qf[t][w]);
            half8_t f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {   // dimension e meets the nibble at bits 4 e: operand slot 2 (e % 4) + e / 4
                const float v = param_scale<E>(x[e >> 1] >> (16 * (e & 1))) * qup;
                f[2 * (e & 3) + (e >> 2)] = (half_t)v;
            }
            qf[t][w] = f;
        }
    }
    const float kscale = p.scale_log2 * pow2(-qe);

    // the wave's steps: [jb, je) in strides of 32 kspl
    const int wi0 = cw / G, wi1 = ncol > 0 ? (cw + ncol - 1) / G : 0;
    const int whi = ncol <= 0 ? 0 : p.causal ? min(k1, max(0, first + wi1 + 1)) : k1;
    const int wlo = p.window ? max(k0, max(0, first + wi0 - p.window + 1) & ~(KV4_TILE - 1)) : k0;
    // steps within [all_lo, all_hi) are seen whole by every column
    const int all_hi = p.causal ? min(len, first + wi0 + 1) : len;
    const int all_lo = p.window ? first + wi1 - p.window + 1 : 0;
    const int stride = KV4_TILE << kshift;
    int j = wlo + KV4_TILE * (wave & (kspl - 1));

    const int32_t* table = p.table + (size_t)b * p.pages_per_seq;
    const int bshift = p.page_shift - 4, last_block = (len - 1) >> 4;
    const size_t page_bytes = (size_t)p.Hkv * kv4_block_bytes(D) << bshift;
    const unsigned char* heads = p.cache + ((size_t)h * kv4_block_bytes(D) << bshift);
    auto page_of = [&](int blk) { return table[min(blk, last_block) >> bshift]; };
    auto block_at = [&](int page, int blk) {
        return heads + (size_t)page * page_bytes + (size_t)(min(blk, last_block) & ((1 << bshift) - 1)) * kv4_block_bytes(D);
    };

    float4_t o[NT][VT];
    float m[NT], l[NT], raise[NT];   // raise: -infinity until a column has seen a key
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = l[t] = 0.f;
        raise[t] = -INFINITY;
#pragma unroll
        for (int x = 0; x < VT; ++x) o[t][x] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    float sref = 0.f, vscale = 0.f;   // a power of two above the largest value scale so far; the weights' factor

    KvTile<D> cur, nxt;
    int bad = 0, bad_n = 0;           // bit s: block s lies in no page
    auto fetch = [&](KvTile<D>& to, int& flags, int at) {
        const int ba = at >> 4, pa = page_of(ba), pb = page_of(ba + 1);
        const bool oa = (unsigned)pa < (unsigned)p.num_pages, ob = (unsigned)pb < (unsigned)p.num_pages;
        load_tile<D>(to, block_at(oa ? pa : 0, ba), block_at(ob ? pb : 0, ba + 1), lane);
        flags = (oa ? 0 : 1) | (ob ? 0 : 2);
    };
    if (j < whi) fetch(cur, bad, j);
    while (j < whi) {
        const int jn = j + stride;
        if (jn < whi) fetch(nxt, bad_n, jn);
        const bool whole = j >= all_lo && j + KV4_TILE <= all_hi && j + KV4_TILE <= whi && !bad;
        if (!whole) {
            // tokens that no column sees may hold anything: their parameters become zeros
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (((bad >> s) & 1) || j + 16 * s + 4 * kb + i >= whi) cur.kp[s][i] = cur.vp[s][i] = 0u;
        }

        float4_t acc[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = float4_t{0.f, 0.f, 0.f, 0.f};
        half2_t kz1[2], kz16[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t z = perm(0u, cur.kc[s], 0x03020302u) & 0x000F000Fu;   // (an unwritten token may hold anything)
            kz1[s] = zero1024(z);
            kz16[s] = zero64(z);
        }
#pragma unroll
        for (int w = 0; w < KW; ++w)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint32_t x = cur.k[s][w], y = x >> 8;
                const half8_t a = as_h8(centred(x, kz1[s]), centred16(x, kz16[s]), centred(y, kz1[s]), centred16(y, kz16[s]));
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[t][s] = mfma16x16x32(a, qf[t][w], acc[t][s]);
            }
        float ks[2][4], vs[2][4], vmax = 0.f;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ks[s][i] = param_scale<E>(cur.kp[s][i]) * kscale;
                vs[s][i] = param_scale<E>(cur.vp[s][i]);
                vmax = fmaxf(vmax, vs[s][i]);
            }
        if (__any(vmax > sref)) {   // rare after the first steps
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) vmax = fmaxf(vmax, __shfl_xor(vmax, x));
            // 2 to 4 times the largest, at least 2^-113 so that the weights' factor stays finite
            const int e = min(126, max(-113, (int)(__float_as_uint(vmax) >> 23) - 127 + 2));
            const float fall = sref * pow2(-e);
            sref = pow2(e);
            vscale = pow2(WEIGHT_LOG2 - e);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int x = 0; x < VT; ++x) o[t][x] *= fall;
            }
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) vs[s][i] *= vscale;
        half8_t pw[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float x[2][4], top = -INFINITY;   // logits less m
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[s][i] = __builtin_fmaf(acc[t][s][i], ks[s][i], -m[t]);
                    if (!whole) {
                        const int at = j + 16 * s + 4 * kb + i;
                        if (at < lo[t] || at >= hi[t] || at >= whi || ((bad >> s) & 1)) x[s][i] = -INFINITY;
                    }
                    top = fmaxf(top, x[s][i]);
                }
            if (__any(top > raise[t])) {
                top = kb_max(top);
                const bool up = top > raise[t];
                const float by = up ? top : 0.f;
                // (a column's first keys: nothing summed yet)
                const float fall = raise[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(-by);
                m[t] += by;
                l[t] *= fall;
#pragma unroll
                for (int y = 0; y < VT; ++y) o[t][y] *= fall;
                if (up) raise[t] = RAISE;
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[s][i] -= by;
            }
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float pj = __builtin_amdgcn_exp2f(x[s][i]);
                    l[t] += pj;
                    // (a token that this column does not see may have a scale of NaN)
                    pw[t][4 * s + i] = (half_t)(!whole && pj == 0.f ? 0.f : pj * vs[s][i]);
                }
        }
        // values: a result tile a nibble
        half2_t vz1[4], vz16[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const uint32_t z = perm(cur.vp[y >> 1][2 * (y & 1) + 1], cur.vp[y >> 1][2 * (y & 1)], 0x07060302u) & 0x000F000Fu;
            vz1[y] = zero1024(z);
            vz16[y] = zero64(z);
        }
#pragma unroll
        for (int g = 0; g < D / 64; ++g) {
            const uint32_t w[4] = {cur.v[0][g], cur.v[0][D / 64 + g], cur.v[1][g], cur.v[1][D / 64 + g]};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                half2_t c[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const uint32_t x = e & 2 ? w[y] >> 8 : w[y];
                    c[y] = e & 1 ? centred16(x, vz16[y]) : centred(x, vz1[y]);
                }
                const half8_t a = as_h8(c[0], c[1], c[2], c[3]);
#pragma unroll
                for (int t = 0; t < NT; ++t) o[t][4 * g + e] = mfma16x16x32(a, pw[t], o[t][4 * g + e]);
            }
        }
        cur = nxt;
        bad = bad_n;
        j = jn;
    }

    // a lane has, of column `col`, dimensions (4 kb + i) D / 16 + x in o[t][x][i]: undo the scales
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        l[t] = kb_sum(l[t]);
        if (raise[t] == -INFINITY && l[t] == 0.f) m[t] = -FLT_MAX;
#pragma unroll
        for (int x = 0; x < VT; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[t][x][i] *= sref * pow2(-WEIGHT_LOG2);
    }
    float *part = nullptr, *part_ml = nullptr;   // this chunk's results and (m, l), by column of the workgroup
    uint32_t* counter = nullptr;
    const size_t slot_floats = (size_t)p.slot_cols * (D + 2);
    float* item = nullptr;
    if (chunks > 1) {
        const size_t at = ((size_t)tile * p.B + b) * p.Hkv + h;
        counter = p.counters + at;
        item = p.partials + at * p.splits * slot_floats;
        part = item + split * slot_floats;
        part_ml = part + (size_t)p.slot_cols * D;
    }
    // four values of column r (of the sequence) from dimension d on
    auto put = [&](int r, int d, float4_t v, float inv) {
        if (chunks > 1) {
            st_partial4<SCOPE_DEVICE>(part + (size_t)(r - c0) * D + d, v);
        } else {
            const int i = r / G;
            uint16_t* dst = static_cast<uint16_t*>(p.out) + (size_t)(q0 + i) * p.o_st + (size_t)(h * G + r - i * G) * p.o_sh + d;
            *reinterpret_cast<u32x2*>(dst) = u32x2{pack2(E{}, saturate<E>(v[0] * inv), saturate<E>(v[1] * inv)),
                                                   pack2(E{}, saturate<E>(v[2] * inv), saturate<E>(v[3] * inv))};
        }
    };
    auto put_ml = [&](int r, float mm, float ll) {
        if (chunks > 1) {
            st_partial<SCOPE_DEVICE>(part_ml + 2 * (r - c0), mm);
            st_partial<SCOPE_DEVICE>(part_ml + 2 * (r - c0) + 1, ll);
        } else if (p.lse) {
            const int i = r / G;
            p.lse[(size_t)(q0 + i) * p.Hq + h * G + r - i * G] = lse_of(mm, ll);
        }
    };
    if (kspl == 1) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int c = 16 * t + col;
            if (c >= ncol) continue;
            const float inv = l[t] == 0.f ? 0.f : 1.f / l[t];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int x = 0; x < VT; x += 4)
                    put(cw + c, (4 * kb + i) * VT + x, float4_t{o[t][x][i], o[t][x + 1][i], o[t][x + 2][i], o[t][x + 3][i]}, inv);
            if (kb == 0) put_ml(cw + c, m[t], l[t]);
        }
    } else {
        // the waves of a group join their shares of the keys
        const int g0 = wave & ~(kspl - 1);
#pragma unroll
        for (int t = 0; t < NT; ++t)
            if (kb == 0) {
                ml[wave][16 * t + col][0] = m[t];
                ml[wave][16 * t + col][1] = l[t];
            }
        __syncthreads();
        const int u = threadIdx.x & (64 * kspl - 1);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float top = ml[g0][16 * t + col][0];
            for (int w = 1; w < kspl; ++w) top = fmaxf(top, ml[g0 + w][16 * t + col][0]);
            const float f = __builtin_amdgcn_exp2f(m[t] - top);
            if (t) __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int x = 0; x < VT; x += 4)
                    *reinterpret_cast<float4_t*>(&red[wave][col * ROW + (4 * kb + i) * VT + x]) =
                        float4_t{o[t][x][i], o[t][x + 1][i], o[t][x + 2][i], o[t][x + 3][i]} * f;
            __syncthreads();
            const int live = min(16, ncol - 16 * t);
            for (int e = u; e < live * (D / 4); e += 64 * kspl) {
                const int c = e / (D / 4), d = 4 * (e - c * (D / 4));
                float mm = ml[g0][16 * t + c][0], ll = 0.f;
                for (int w = 1; w < kspl; ++w) mm = fmaxf(mm, ml[g0 + w][16 * t + c][0]);
                float4_t v = {0.f, 0.f, 0.f, 0.f};
                for (int w = 0; w < kspl; ++w) {
                    ll += ml[g0 + w][16 * t + c][1] * __builtin_amdgcn_exp2f(ml[g0 + w][16 * t + c][0] - mm);
                    v += *reinterpret_cast<const float4_t*>(&red[g0 + w][c * ROW + d]);
                }
                put(cw + 16 * t + c, d, v, ll == 0.f ? 0.f : 1.f / ll);
                if (d == 0) put_ml(cw + 16 * t + c, mm, ll);
            }
        }
    }
    if (chunks == 1) return;

    // the last chunk to arrive joins them, in order
    if (!splitk_arrive(counter, chunks, &last)) return;
    const int live = min(4 * COLS, cols);
    for (int e = threadIdx.x; e < live * (D / 4); e += 256) {
        const int c = e / (D / 4), d = 4 * (e - c * (D / 4));
        const float* at = item + (size_t)p.slot_cols * D + 2 * c;
        float mm = -FLT_MAX;
        for (int s = 0; s < chunks; ++s) mm = fmaxf(mm, __hip_atomic_load(at + s * slot_floats, __ATOMIC_RELAXED, SCOPE_DEVICE));
        float ll = 0.f;
        float4_t v = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < chunks; ++s) {
            const float f = __builtin_amdgcn_exp2f(__hip_atomic_load(at + s * slot_floats, __ATOMIC_RELAXED, SCOPE_DEVICE) - mm);
            ll += f * __hip_atomic_load(at + s * slot_floats + 1, __ATOMIC_RELAXED, SCOPE_DEVICE);
            v += ld_partial4<SCOPE_DEVICE>(item + s * slot_floats + (size_t)c * D + d) * f;
        }
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        const int r = c0 + c, i = r / G;
        uint16_t* dst = static_cast<uint16_t*>(p.out) + (size_t)(q0 + i) * p.o_st + (size_t)(h * G + r - i * G) * p.o_sh + d;
        *reinterpret_cast<u32x2*>(dst) = u32x2{pack2(E{}, saturate<E>(v[0] * inv), saturate<E>(v[1] * inv)),
                                               pack2(E{}, saturate<E>(v[2] * inv), saturate<E>(v[3] * inv))};
        if (d == 0 && p.lse) p.lse[(size_t)(q0 + i) * p.Hq + h * G + r - i * G] = lse_of(mm, ll);
    }
}

Kv4AttnShape kv4_attention_shape(int T, int B, int Hq, int Hkv, int D, int max_q, int max_kv, int num_cus) {
    Kv4AttnShape s{};
    const int64_t G = Hq / Hkv, C = (int64_t)(max_q < T ? max_q : T) * G;
    s.nt = D <= 128 && C > 16 ? 2 : 1;
    const int wg_cols = 64 * s.nt;
    const int64_t tiles = std::max<int64_t>(1, (C + wg_cols - 1) / wg_cols), items = tiles * B * Hkv;
    const int64_t target = 2 * num_cus;
    auto chunk_of = [&](int64_t least, int64_t most) {
        const int64_t c = ((int64_t)max_kv * items / target + 127) / 128 * 128;
        return (int)std::min(std::max(c, least), most);
    };
    s.chunk_thin = chunk_of(128, 2048);
    s.chunk_full = items >= target ? (INT32_MAX / 2) & ~127 : chunk_of(256, 1 << 24);
    const bool full = C > wg_cols / 2;
    const int least = full ? std::min(s.chunk_thin, s.chunk_full) : s.chunk_thin;
    s.splits = max_kv <= least ? 1 : (int)(((int64_t)max_kv + least - 1) / least);
    if (items > (int64_t)KV4_MAX_COUNTERS) s.splits = 1;
    s.ok = tiles * s.splits <= 65535;
    s.tiles = (int)std::min<int64_t>(tiles, 65535);
    s.slot_cols = (int)std::min<int64_t>(wg_cols, (C + 15) / 16 * 16);
    if (s.splits > 1) s.partial_bytes = (size_t)items * s.splits * s.slot_cols * (D + 2) * sizeof(float);
    return s;
}

template <typename E, int D>
static void go(const Kv4AttnShape& s, const Kv4AttnParams& p, hipStream_t st) {
    const dim3 grid(p.Hkv, p.B, s.tiles * s.splits);
    if constexpr (D <= 128)
        if (s.nt == 2) {
            kv4_attention_kernel<E, D, 2><<<grid, 256, 0, st>>>(p);
            return;
        }
    kv4_attention_kernel<E, D, 1><<<grid, 256, 0, st>>>(p);
}

hipError_t launch_kv4_attention(bool bf16, int D, Kv4AttnParams p, const Kv4AttnShape& s, hipStream_t st) {
    p.G = p.Hq / p.Hkv;
    p.tiles = s.tiles; p.splits = s.splits; p.chunk_thin = s.chunk_thin; p.chunk_full = s.chunk_full;
    p.slot_cols = s.slot_cols;
    switch (D) {
        case 64: bf16 ? go<bf16_t, 64>(s, p, st) : go<half_t, 64>(s, p, st); break;
        case 128: bf16 ? go<bf16_t, 128>(s, p, st) : go<half_t, 128>(s, p, st); break;
        case 192: bf16 ? go<bf16_t, 192>(s, p, st) : go<half_t, 192>(s, p, st); break;
        case 256: bf16 ? go<bf16_t, 256>(s, p, st) : go<half_t, 256>(s, p, st); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace w4a16
