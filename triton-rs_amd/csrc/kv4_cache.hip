// Rows of keys and values into the 4-bit cache (kv4.h), and back.
//
// A row x[0, D) of one token and head: s = RNE_E(f32((max - min) / 15)) over the range that it and 0
// span, z = rint(-min / s), n = clamp(rint(x / s) + z, 0, 15), ties to even; s = 0 gives n = z = 0, a
// row with an infinity or NaN s = NaN (it reads back as NaN). Read back: RNE_E((n - z) s), saturated.
//
// Bound by memory: 2 D bytes of a row against D / 2 + 4. A workgroup takes 16 tokens of one head, a
// row 16 lanes of D / 16 dimensions each (a column of the value layout), so a wave's four rows write
// 256 contiguous bytes of keys and of values where their slots are consecutive.
#include "device_common.h"
#include "kv4.h"

namespace w4a16 {

// D / 16 elements of a row, as 8-byte loads and stores
template <int N>
struct Elems { uint32_t w[N / 2]; };

template <int N>
__device__ __forceinline__ Elems<N> load_elems(const void* base, size_t elem) {
    Elems<N> r;
    const u32x2* p = reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(base) + elem);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const u32x2 t = p[i];
        r.w[2 * i] = t[0];
        r.w[2 * i + 1] = t[1];
    }
    return r;
}

template <typename E>
__device__ __forceinline__ float elem_f32(uint32_t bits16) {
    if constexpr (__is_same(E, half_t)) return (float)__builtin_bit_cast(half_t, (uint16_t)bits16);
    else return bf16_bits_to_f32(bits16 & 0xFFFFu);
}
template <typename E>
__device__ __forceinline__ uint32_t elem_bits(float v) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (E)v);
}

// Where a slot's row lies: its block, and its token in the block. false: outside the cache.
__device__ __forceinline__ bool slot_block(const Kv4RowParams& p, int t, int h, int block_bytes, unsigned char** block, int* tok) {
    if (t >= p.T) return false;
    const int slot = p.slots[t];
    const int page = slot >> p.page_shift;
    if (slot < 0 || page >= p.num_pages) return false;
    const int in_page = slot & ((1 << p.page_shift) - 1);
    const int blocks = 1 << (p.page_shift - 4);
    *block = p.cache + ((size_t)((size_t)page * p.Hkv + h) * blocks + (in_page >> 4)) * block_bytes;
    *tok = in_page & 15;
    return true;
}

template <typename E, int D>
__device__ __forceinline__ void quantise_row(const Elems<D / 16>& x, int c, int tok, unsigned char* block, bool is_value) {
    constexpr int N = D / 16;
    float f[N], lo = 0.f, hi = 0.f;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t b = (x.w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu;
        f[i] = elem_f32<E>(b);
        lo = fminf(lo, f[i]);
        hi = fmaxf(hi, f[i]);
        top = max(top, b & 0x7FFFu);
    }
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, m));
        hi = fmaxf(hi, __shfl_xor(hi, m));
        top = max(top, (uint32_t)__shfl_xor((int)top, m));
    }
    const bool finite = top < (__is_same(E, half_t) ? 0x7C00u : 0x7F80u);
    uint32_t sbits = elem_bits<E>((float)(((double)hi - (double)lo) / 15.0));
    const float s = elem_f32<E>(sbits);
    const bool some = finite && s > 0.f;
    const float z = some ? fminf(fmaxf(rintf(-lo / s), 0.f), 15.f) : 0.f;
    if (!finite) sbits = __is_same(E, half_t) ? 0x7E00u : 0x7FC0u;
    uint32_t nib[(N + 7) / 8] = {};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        // x and s have 11 bits at most: x / s is either a tie or further from one than fp32's rounding
        const float n = some ? fminf(fmaxf(rintf(f[i] / s) + z, 0.f), 15.f) : 0.f;
        nib[i >> 3] |= (uint32_t)n << (4 * (i & 7));
    }
    if (!is_value) {
        uint16_t* dst = reinterpret_cast<uint16_t*>(block + tok * (D / 2) + c * (D / 32));
#pragma unroll
        for (int i = 0; i < N / 4; ++i) dst[i] = (uint16_t)(nib[i >> 1] >> (16 * (i & 1)));
    } else {
        unsigned char* dst = block + 8 * D + (tok >> 2) * (2 * D) + c * (D / 8) + ((tok >> 1) & 1) * (D / 16) + 2 * (tok & 1);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) *reinterpret_cast<uint16_t*>(dst + 4 * i) = (uint16_t)(nib[i >> 1] >> (16 * (i & 1)));
    }
    if (c == 0) *reinterpret_cast<uint32_t*>(block + 16 * D + (is_value ? 64 : 0) + 4 * tok) = sbits | ((uint32_t)z << 16);
}

template <typename E, int D>
__global__ __launch_bounds__(256) void kv4_write_kernel(Kv4RowParams p) {
    const int c = threadIdx.x & 15, t = blockIdx.x * 16 + (threadIdx.x >> 4), h = blockIdx.y;
    unsigned char* block;
    int tok;
    // the 16 lanes of a row agree
    if (!slot_block(p, t, h, kv4_block_bytes(D), &block, &tok)) return;
    const Elems<D / 16> k = load_elems<D / 16>(p.k, (size_t)t * p.k_st + (size_t)h * p.k_sh + c * (D / 16));
    const Elems<D / 16> v = load_elems<D / 16>(p.v, (size_t)t * p.v_st + (size_t)h * p.v_sh + c * (D / 16));
    quantise_row<E, D>(k, c, tok, block, false);
    quantise_row<E, D>(v, c, tok, block, true);
}

template <typename E, int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4RowParams p) {
    constexpr int N = D / 16;
    const int c = threadIdx.x & 15, t = blockIdx.x * 16 + (threadIdx.x >> 4), h = blockIdx.y;
    unsigned char* block;
    int tok;
    if (!slot_block(p, t, h, kv4_block_bytes(D), &block, &tok)) return;
    constexpr float most = __is_same(E, half_t) ? 65504.f : 0x1.fep127f;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(block + 16 * D + 64 * kv + 4 * tok);
        const float s = elem_f32<E>(w), z = (float)(w >> 16);
        const unsigned char* src = kv ? block + 8 * D + (tok >> 2) * (2 * D) + c * (D / 8) + ((tok >> 1) & 1) * (D / 16) + 2 * (tok & 1)
                                      : block + tok * (D / 2) + c * (D / 32);
        uint32_t o[N / 2];
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint32_t n4 = *reinterpret_cast<const uint16_t*>(src + (kv ? 4 : 2) * i);
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float r = ((float)((n4 >> (4 * e)) & 15u) - z) * s;
                // (15 s may pass the largest value by less than a step; NaN stays)
                x[e] = r > most ? most : r < -most ? -most : r;
            }
            o[2 * i] = pack2(E{}, x[0], x[1]);
            o[2 * i + 1] = pack2(E{}, x[2], x[3]);
        }
        uint16_t* out = static_cast<uint16_t*>(kv ? p.v_out : p.k_out) +
                        ((size_t)t * (kv ? p.v_st : p.k_st) + (size_t)h * (kv ? p.v_sh : p.k_sh) + c * N);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) reinterpret_cast<u32x2*>(out)[i] = u32x2{o[2 * i], o[2 * i + 1]};
    }
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
