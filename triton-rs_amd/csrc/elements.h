// Rows of 16-bit elements at any element's address, as fp32: shared by the kernels that take rows as they lie.
#pragma once
#include "device_common.h"

namespace w4a16 {

// Eight elements at an address that is aligned to one: global memory takes unaligned vectors, at the rate of
// the lines that they touch.
struct __attribute__((packed, aligned(2))) Elems8 { uint32_t w[4]; };
struct __attribute__((packed, aligned(1))) Bytes8 { uint32_t w[2]; };

template <typename E>
__device__ __forceinline__ float elem_to_f32(uint32_t bits16) {
    if constexpr (__is_same(E, half_t)) return (float)__builtin_bit_cast(half_t, (uint16_t)bits16);
    else return bf16_bits_to_f32(bits16);   // the shift drops the upper half
}
template <typename E>
__device__ __forceinline__ uint32_t f32_to_elem(float v) { return (uint32_t)__builtin_bit_cast(uint16_t, (E)v); }

// Elements [0, n) of eight at p, the others 0.
__device__ __forceinline__ Elems8 load8(const uint16_t* p, int n) {
    Elems8 r = {{0, 0, 0, 0}};
    if (n >= 8) {
        r = *reinterpret_cast<const Elems8*>(p);
    } else if (n > 0) {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < n) r.w[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
    }
    return r;
}
__device__ __forceinline__ void store8(uint16_t* p, const Elems8& v, int n) {
    if (n >= 8) {
        *reinterpret_cast<Elems8*>(p) = v;
    } else if (n > 0) {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < n) p[e] = (uint16_t)(v.w[e >> 1] >> (16 * (e & 1)));
    }
}
template <typename E>
__device__ __forceinline__ void to_f32(const Elems8& v, float (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f[2 * e] = elem_to_f32<E>(v.w[e]);
        if constexpr (__is_same(E, half_t)) f[2 * e + 1] = elem_to_f32<E>(v.w[e] >> 16);
        else f[2 * e + 1] = __uint_as_float(v.w[e] & 0xFFFF0000u);
    }
}
template <typename E>
__device__ __forceinline__ Elems8 from_f32(const float (&f)[8]) {
    Elems8 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v.w[e] = pack2(E{}, f[2 * e], f[2 * e + 1]);
    return v;
}

// v, or the largest finite value of the element type beyond it (NaN stays)
template <typename E>
__device__ __forceinline__ float saturate(float v) {
    constexpr float most = __is_same(E, half_t) ? 65504.f : 0x1.fep127f;
    return v > most ? most : v < -most ? -most : v;
}

// Four fp32 values of at most 448 in magnitude as e4m3 bytes, lowest first, each rounded to nearest even.
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

}  // namespace w4a16
