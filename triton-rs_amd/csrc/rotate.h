// The rotation of a pair of dimensions at a position, as every kernel that rotates computes it.
#pragma once
#include "elements.h"

namespace w4a16 {

// magnitude times (cos, sin) of position * f radians: the angle in whole turns in fp64, its fraction exact.
__device__ __forceinline__ float2 angle(int position, double f, float magnitude) {
    const double turns = (double)position * f * 0.15915494309189533577;   // 1 / (2 pi)
    double s, c;
    sincospi(2.0 * (turns - rint(turns)), &s, &c);
    return float2{(float)(magnitude * c), (float)(magnitude * s)};
}

// (a, b) turned, in fp32: each product is rounded, then their difference or sum (no contraction)
__device__ __forceinline__ void turn_pair(float& a, float& b, float2 w) {
#pragma clang fp contract(off)
    const float x = a * w.x - b * w.y, y = a * w.y + b * w.x;
    a = x;
    b = y;
}
// the same, to the element type's largest finite value beyond that
template <typename E>
__device__ __forceinline__ void rotate(float& a, float& b, float2 w) {
    turn_pair(a, b, w);
    a = saturate<E>(a);
    b = saturate<E>(b);
}

// Unit u of a row: the first `turned` of them are eight elements (PAIRS), or eight and their eight partners; the others
// are eight each of those beyond rot, which are copied. o may be x.
template <typename E, bool PAIRS>
__device__ __forceinline__ void turn_unit(const uint16_t* x, uint16_t* o, const float2* a, int u, int turned, int rot, int D) {
    const int half = rot / 2;
    if (u >= turned) {
        const int e = rot + 8 * (u - turned);
        if (x != o) store8(o + e, load8(x + e, D - e), D - e);
    } else if constexpr (PAIRS) {
        float f[8];
        to_f32<E>(load8(x + 8 * u, rot - 8 * u), f);
#pragma unroll
        for (int i = 0; i < 4; ++i) rotate<E>(f[2 * i], f[2 * i + 1], a[min(4 * u + i, half - 1)]);
        store8(o + 8 * u, from_f32<E>(f), rot - 8 * u);
    } else {
        float f[8], g[8];
        to_f32<E>(load8(x + 8 * u, half - 8 * u), f);
        to_f32<E>(load8(x + half + 8 * u, half - 8 * u), g);
#pragma unroll
        for (int i = 0; i < 8; ++i) rotate<E>(f[i], g[i], a[min(8 * u + i, half - 1)]);
        store8(o + 8 * u, from_f32<E>(f), half - 8 * u);
        store8(o + half + 8 * u, from_f32<E>(g), half - 8 * u);
    }
}
__host__ __device__ constexpr int turned_units(int rot, bool pairs) { return pairs ? (rot + 7) / 8 : (rot / 2 + 7) / 8; }
__host__ __device__ constexpr int row_units(int rot, int D, bool pairs) { return turned_units(rot, pairs) + (D - rot + 7) / 8; }

}  // namespace w4a16
