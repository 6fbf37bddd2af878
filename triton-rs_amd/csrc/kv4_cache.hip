// Rows of keys and values into the 4-bit cache (kv4.h), and back.
//
// A row x[0, D) of one token and head: s = RNE_E(f32((max - min) / 15)) over the range that it and 0
// span, z = rint(-min / s), n = clamp(rint(x / s) + z, 0, 15), ties to even; s = 0 gives n = z = 0, a
// row with an infinity or NaN s = NaN (it reads back as NaN). Read back: RNE_E((n - z) s), saturated.
//
// Bound by memory: 2 D bytes of a row against D / 2 + 4. A workgroup takes 16 tokens of one head, a
// row 16 lanes of D / 16 dimensions each (a column of the value layout), so a wave's four rows write
// 256 contiguous bytes of keys and of values where their slots are consecutive. Vector instructions are
// kept to about 18 an element, addresses included (writing; division, conversion and clamping one by one took twice as
// long as the memory): extremes as ordered 16-bit integers in pairs, and x / s rounded by two additions.
// Measured, bf16, 8 heads of D = 128: 8192 tokens written in 12.1 us (3.5 TB/s), read back in 9.6 (4.4); 65536
// read in 78 (4.4; a large copy reaches 4.8). A few rows take 3 us a kernel, 7 a call.
#include "device_common.h"
#include "kv4.h"

namespace w4a16 {

template <typename E>
__device__ __forceinline__ float elem_f32(uint32_t bits16) {
    if constexpr (__is_same(E, half_t)) return (float)__builtin_bit_cast(half_t, (uint16_t)bits16);
    else return bf16_bits_to_f32(bits16);   // the shift drops the upper half
}
template <typename E>
__device__ __forceinline__ uint32_t elem_bits(float v) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (E)v);
}
template <typename E>
constexpr int INF_BITS = __is_same(E, half_t) ? 0x7C00 : 0x7F80;

typedef short short2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ short2_t as_s2(uint32_t u) { return __builtin_bit_cast(short2_t, u); }

// A lane's N = D / 16 elements of a row.
template <int N>
struct Elems { uint32_t w[N / 2]; };

template <int N>
__device__ __forceinline__ Elems<N> load_elems(const void* base, size_t elem) {
    Elems<N> r;
    const uint16_t* p = static_cast<const uint16_t*>(base) + elem;
    if constexpr (N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) {
            const u32x4 t = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) r.w[4 * i + e] = t[e];
        }
    } else {   // (24 bytes a lane are 8-byte aligned)
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const u32x2 t = reinterpret_cast<const u32x2*>(p)[i];
            r.w[2 * i] = t[0];
            r.w[2 * i + 1] = t[1];
        }
    }
    return r;
}

template <int N>
__device__ __forceinline__ void store_elems(void* base, size_t elem, const uint32_t (&w)[N / 2]) {
    uint16_t* p = static_cast<uint16_t*>(base) + elem;
    if constexpr (N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) reinterpret_cast<u32x4*>(p)[i] = u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) reinterpret_cast<u32x2*>(p)[i] = u32x2{w[2 * i], w[2 * i + 1]};
    }
}

// Where a slot's row lies: its block, and its token in the block. false: outside the cache.
__device__ __forceinline__ bool slot_block(const Kv4RowParams& p, int slot, int h, int block_bytes, unsigned char** block, int* tok) {
    const int page = slot >> p.page_shift;
    if (slot < 0 || page >= p.num_pages) return false;
    const int in_page = slot & ((1 << p.page_shift) - 1);
    *block = p.cache + (((((size_t)page * p.Hkv + h) << (p.page_shift - 4)) + (in_page >> 4)) * block_bytes);
    *tok = in_page & 15;
    return true;
}
// This lane's bytes of a token's values: D / 64 words of 16 bits, 4 bytes apart.
template <int D>
__device__ __forceinline__ unsigned char* value_words(unsigned char* block, int tok, int c) {
    return block + 8 * D + (tok >> 2) * (2 * D) + c * (D / 8) + ((tok >> 1) & 1) * (D / 16) + 2 * (tok & 1);
}

// Smallest (at most 0) and largest (at least 0) of a row over its 16 lanes, as ordered integers: the element's
// bits, those of negative ones but the sign inverted. An infinity or NaN lies beyond +-INF_BITS.
struct Extremes { int lo, hi; };
template <int N>
__device__ __forceinline__ Extremes extremes(const Elems<N>& x) {
    short2_t lo = {0, 0}, hi = {0, 0};
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const short2_t b = as_s2(x.w[i]);
        const short2_t o = b ^ ((b >> (short)15) & (short)0x7FFF);
        lo = __builtin_elementwise_min(lo, o);
        hi = __builtin_elementwise_max(hi, o);
    }
    Extremes r = {min((int)lo[0], (int)lo[1]), max((int)hi[0], (int)hi[1])};
    // lanes of a row of 16: neighbours, pairs, halves mirrored, the row mirrored
#define KV4_STEP(ctrl)                                                              \
    r.lo = min(r.lo, __builtin_amdgcn_update_dpp(r.lo, r.lo, ctrl, 0xF, 0xF, true)); \
    r.hi = max(r.hi, __builtin_amdgcn_update_dpp(r.hi, r.hi, ctrl, 0xF, 0xF, true))
    KV4_STEP(0xB1);
    KV4_STEP(0x4E);
    KV4_STEP(0x141);
    KV4_STEP(0x140);
#undef KV4_STEP
    return r;
}
__device__ __forceinline__ uint32_t ordered_bits(int o) { return (uint32_t)(o < 0 ? o ^ 0x7FFF : o) & 0xFFFFu; }

// Bits of s = RNE_E(f32(d / 15)), d = hi - lo. The quotient is that of fp64's division: q + r / 15 with the
// remainder r of a first q exact (fma) rounds correctly.
template <typename E>
__device__ __forceinline__ uint32_t scale_bits(float lo, float hi) {
    const double d = (double)hi - (double)lo, inv = 1.0 / 15.0, q = d * inv;
    return elem_bits<E>((float)__builtin_fma(__builtin_fma(-15.0, q, d), inv, q));
}

// The row's parameters and this lane's nibbles, lowest dimension first.
//
// rint(x / s), ties to even: x and s have 11 significant bits at most, so a quotient of at most 15.5 that is no
// tie is at least 2^-12 away from one. t = fma(x, 1/s, 1536) rounds it to a multiple of 2^-13 (the
// reciprocal's error of some 2^-19 is not seen), a tie to the tie itself; t + (M - 1536), M = 1.5 2^23,
// rounds that to an integer, ties to even, in the low bits of M + rint(x / s).
template <typename E, int N>
__device__ __forceinline__ uint32_t quantise(const Elems<N>& x, Extremes r, uint32_t sbits, uint32_t (&word)[(N + 7) / 8]) {
    constexpr float FINE = 1536.f, M = 12582912.f;
    constexpr uint32_t M_BITS = 0x4B400000u;
    const bool finite = r.hi < INF_BITS<E> && r.lo > -INF_BITS<E> - 1;
    float s = elem_f32<E>(sbits), up = 1.f;
    const bool some = finite && s > 0.f;
    if constexpr (!__is_same(E, half_t)) {   // a reciprocal of 2^-126 and less overflows
        if (s < 0x1p-60f) {
            up = 0x1p60f;
            s *= up;
        }
    }
    const float inv = some ? __builtin_amdgcn_rcpf(s) : 0.f;
    const float lo = some ? elem_f32<E>(ordered_bits(r.lo)) : 0.f;
    const float z = fminf((__builtin_fmaf(-lo * up, inv, FINE) + (M - FINE)) - M, 15.f);   // (-lo is not negative)
    const float least = M - z, most = M + 15.f - z;
    const uint32_t zi = (uint32_t)z;
#pragma unroll
    for (int g = 0; g < (N + 7) / 8; ++g) {
        uint32_t acc = 0, bias = 0;
#pragma unroll
        for (int i = 7; i >= 0; --i) {
            const int e = 8 * g + i;
            if (e >= N) continue;
            float v = elem_f32<E>(x.w[e >> 1] >> (16 * (e & 1)));
            if constexpr (!__is_same(E, half_t)) v *= up;
            const float n = __builtin_amdgcn_fmed3f(__builtin_fmaf(v, inv, FINE) + (M - FINE), least, most);
            acc = (acc << 4) + __float_as_uint(n);
            bias = (bias << 4) + M_BITS;
        }
        // M's bits out, the zero point added to every nibble (each sum is 0..15)
        word[g] = some ? acc - bias + zi * (N - 8 * g >= 8 ? 0x11111111u : 0x1111u) : 0u;
    }
    return (finite ? sbits : __is_same(E, half_t) ? 0x7E00u : 0x7FC0u) | zi << 16;
}

template <typename E, int D>
__global__ __launch_bounds__(256) void kv4_write_kernel(Kv4RowParams p) {
    constexpr int N = D / 16;
    const int c = threadIdx.x & 15, t = blockIdx.x * 16 + (threadIdx.x >> 4), h = blockIdx.y;
    if (t >= p.T) return;   // (the 16 lanes of a row agree, here and below)
    const int slot = p.slots[t];
    const Elems<N> k = load_elems<N>(p.k, (size_t)t * p.k_st + (size_t)h * p.k_sh + c * N);
    const Elems<N> v = load_elems<N>(p.v, (size_t)t * p.v_st + (size_t)h * p.v_sh + c * N);
    unsigned char* block;
    int tok;
    if (!slot_block(p, slot, h, kv4_block_bytes(D), &block, &tok)) return;
    const Extremes rk = extremes(k), rv = extremes(v);
    // half a row's lanes divide for the keys, half for the values
    const bool lower = c < 8;
    const uint32_t mine = scale_bits<E>(elem_f32<E>(ordered_bits(lower ? rk.lo : rv.lo)), elem_f32<E>(ordered_bits(lower ? rk.hi : rv.hi)));
    const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)mine, 0x128, 0xF, 0xF, true);   // 8 lanes round the row
    uint32_t wk[(N + 7) / 8], wv[(N + 7) / 8];
    const uint32_t pk = quantise<E, N>(k, rk, lower ? mine : other, wk);
    const uint32_t pv = quantise<E, N>(v, rv, lower ? other : mine, wv);
    unsigned char* dk = block + tok * (D / 2) + c * (D / 32);
    if constexpr (D == 128) *reinterpret_cast<uint32_t*>(dk) = wk[0];
    else if constexpr (D == 256) *reinterpret_cast<u32x2*>(dk) = u32x2{wk[0], wk[1]};
    else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) reinterpret_cast<uint16_t*>(dk)[i] = (uint16_t)(wk[i >> 1] >> (16 * (i & 1)));
    }
    unsigned char* dv = value_words<D>(block, tok, c);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) *reinterpret_cast<uint16_t*>(dv + 4 * i) = (uint16_t)(wv[i >> 1] >> (16 * (i & 1)));
    if (c < 2) *reinterpret_cast<uint32_t*>(block + 16 * D + 64 * c + 4 * tok) = c ? pv : pk;
}

// Eight nibbles as RNE_E((n - z) s) in four words. fp16: n - z is exact, so one fp16 product rounds once; bf16:
// (n - z) s is exact in fp32. Where 15 s passes the largest finite value (by less than a step) the result is that.
template <typename E>
__device__ __forceinline__ void dequantise8(uint32_t x, uint32_t par, uint32_t (&o)[4]) {
    const float s = elem_f32<E>(par);
    if constexpr (__is_same(E, half_t)) {
        const uint32_t z = perm(0u, par, 0x03020302u), y = x >> 8;
        const half2_t z1 = as_h2(z | 0x64006400u), z16 = as_h2((z << 4) | 0x54005400u), sixteenth = {(half_t)0.0625f, (half_t)0.0625f};
        const half2_t s2 = as_h2(perm(0u, par, 0x01000100u));
        half2_t a[4] = {nib_pair(x) - z1, __builtin_elementwise_fma(nib_pair16(x), sixteenth, -z16), nib_pair(y) - z1,
                        __builtin_elementwise_fma(nib_pair16(y), sixteenth, -z16)};   // (0, 4), (1, 5), (2, 6), (3, 7)
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] *= s2;
        if (s > 4096.f) {
            const half2_t most = {(half_t)65504.f, (half_t)65504.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = __builtin_elementwise_max(__builtin_elementwise_min(a[i], most), -most);
        }
        o[0] = perm(as_u32(a[1]), as_u32(a[0]), 0x05040100u);
        o[1] = perm(as_u32(a[3]), as_u32(a[2]), 0x05040100u);
        o[2] = perm(as_u32(a[1]), as_u32(a[0]), 0x07060302u);
        o[3] = perm(as_u32(a[3]), as_u32(a[2]), 0x07060302u);
    } else {
        // (z s may pass fp32 where (n - z) s does not; the bound of a row of NaN is NaN, and so is the middle of three)
        const float z = (float)(par >> 16), most = s == s ? 0x1.fep127f : s;
        float f[8];
        auto value = [&](uint32_t n) { return __builtin_amdgcn_fmed3f(((float)n - z) * s, -most, most); };
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // bytes: nibbles 2 i and 2 i + 1
            f[2 * i] = value(((x & 0x0F0F0F0Fu) >> (8 * i)) & 0xFFu);
            f[2 * i + 1] = value((((x >> 4) & 0x0F0F0F0Fu) >> (8 * i)) & 0xFFu);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = pack2(E{}, f[2 * i], f[2 * i + 1]);
    }
}

template <typename E, int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4RowParams p) {
    constexpr int N = D / 16, W = (N + 7) / 8;
    const int c = threadIdx.x & 15, t = blockIdx.x * 16 + (threadIdx.x >> 4), h = blockIdx.y;
    unsigned char* block;
    int tok;
    if (t >= p.T || !slot_block(p, p.slots[t], h, kv4_block_bytes(D), &block, &tok)) return;
    const uint32_t pk = *reinterpret_cast<const uint32_t*>(block + 16 * D + 4 * tok), pv = *reinterpret_cast<const uint32_t*>(block + 16 * D + 64 + 4 * tok);
    const unsigned char *sk = block + tok * (D / 2) + c * (D / 32), *sv = value_words<D>(block, tok, c);
    uint32_t wk[W] = {}, wv[W] = {};
    if constexpr (D == 128) wk[0] = *reinterpret_cast<const uint32_t*>(sk);
    else if constexpr (D == 256) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(sk);
        wk[0] = x[0];
        wk[1] = x[1];
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) wk[i >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(sk)[i] << (16 * (i & 1));
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) wv[i >> 1] |= (uint32_t)*reinterpret_cast<const uint16_t*>(sv + 4 * i) << (16 * (i & 1));
    uint32_t ok[4 * W], ov[4 * W];
#pragma unroll
    for (int g = 0; g < W; ++g) {
        uint32_t a[4], b[4];
        dequantise8<E>(wk[g], pk, a);
        dequantise8<E>(wv[g], pv, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ok[4 * g + i] = a[i];
            ov[4 * g + i] = b[i];
        }
    }
    uint32_t rk[N / 2], rv[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        rk[i] = ok[i];
        rv[i] = ov[i];
    }
    store_elems<N>(p.k_out, (size_t)t * p.k_st + (size_t)h * p.k_sh + c * N, rk);
    store_elems<N>(p.v_out, (size_t)t * p.v_st + (size_t)h * p.v_sh + c * N, rv);
}

template <template <typename, int> class K>
static hipError_t launch_rows(bool bf16, int D, const Kv4RowParams& p, hipStream_t st) {
    const dim3 grid((p.T + 15) / 16, p.Hkv);
    switch (D) {
        case 64: bf16 ? K<bf16_t, 64>::go(grid, p, st) : K<half_t, 64>::go(grid, p, st); break;
        case 128: bf16 ? K<bf16_t, 128>::go(grid, p, st) : K<half_t, 128>::go(grid, p, st); break;
        case 192: bf16 ? K<bf16_t, 192>::go(grid, p, st) : K<half_t, 192>::go(grid, p, st); break;
        case 256: bf16 ? K<bf16_t, 256>::go(grid, p, st) : K<half_t, 256>::go(grid, p, st); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

template <typename E, int D>
struct WriteRows {
    static void go(dim3 grid, const Kv4RowParams& p, hipStream_t st) { kv4_write_kernel<E, D><<<grid, 256, 0, st>>>(p); }
};
template <typename E, int D>
struct ReadRows {
    static void go(dim3 grid, const Kv4RowParams& p, hipStream_t st) { kv4_read_kernel<E, D><<<grid, 256, 0, st>>>(p); }
};

hipError_t launch_kv4_write(bool bf16, int D, const Kv4RowParams& p, hipStream_t st) { return launch_rows<WriteRows>(bf16, D, p, st); }
hipError_t launch_kv4_read(bool bf16, int D, const Kv4RowParams& p, hipStream_t st) { return launch_rows<ReadRows>(bf16, D, p, st); }

}  // namespace w4a16
