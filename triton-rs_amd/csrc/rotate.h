// The rotation of a pair of dimensions at a position, as every kernel that rotates computes it.
#pragma once
#include "elements.h"

namespace w4a16 {

// magnitude times (cos, sin) of position * f radians in fp32, off by 0.76 units at most (8 million angles of up to 2 10^6 radians) where
// that is 0.05 or more; next to zero the angle's rounding in fp64, 2^-53 of it, counts.
//
// The angle in whole turns in fp64, its fraction exact; the nearest quarter turn n off it leaves y in [-pi / 4, pi / 4],
// taken as a sum of two fp32 numbers. Sine and cosine of that are Taylor's series to y^11 and y^10 (remainders below 2^-37
// and 2^-33) with their leading terms, y and 1 - y^2 / 2, kept apart from the rest. Some 13
// fp64 and 30 fp32 instructions; sincospi in fp64 and its rounding made an appended prompt's launch 10% longer.
__device__ __forceinline__ float2 angle(int position, double f, float magnitude) {
#pragma clang fp contract(off)   // (the same bits in every kernel)
    const double turns = (double)position * f * 0.15915494309189533577;   // 1 / (2 pi)
    const double part = turns - rint(turns), quarter = rint(4.0 * part);
    const double y = __builtin_fma(quarter, -0.25, part) * 6.28318530717958647693;
    const float h = (float)y, low = (float)(y - (double)h);
    const float q = h * h, e = __builtin_fmaf(h, h, -q);
    auto poly = [q](float a, float b, float c, float d) { return __builtin_fmaf(q, __builtin_fmaf(q, __builtin_fmaf(q, d, c), b), a); };
    // sin = h + sin_rest, cos = c + cos_rest
    const float ps = q * __builtin_fmaf(q, poly(1.f / 120, -1.f / 5040, 1.f / 362880, -1.f / 39916800), -1.f / 6);
    const float sin_rest = __builtin_fmaf(h, ps, low * __builtin_fmaf(q, -0.5f, 1.f));
    const float pc = q * q * poly(1.f / 24, -1.f / 720, 1.f / 40320, -1.f / 3628800);
    const float c = __builtin_fmaf(q, -0.5f, 1.f), lost = __builtin_fmaf(q, -0.5f, 1.f - c);
    const float cos_rest = pc + (lost - __builtin_fmaf(h, low, 0.5f * e));
    const float sine = __builtin_fmaf(magnitude, h, magnitude * sin_rest), cosine = __builtin_fmaf(magnitude, c, magnitude * cos_rest);
    const int n = (int)quarter & 3;
    const float x = n & 1 ? sine : cosine, z = n & 1 ? cosine : sine;
    return float2{n == 1 || n == 2 ? -x : x, n >= 2 ? -z : z};
}

// (a, b) turned, in fp32: each product is rounded, then their difference or sum (no contraction)
__device__ __forceinline__ void turn_pair(float& a, float& b, float2 w) {
#pragma clang fp contract(off)
    const float x = a * w.x - b * w.y, y = a * w.y + b * w.x;
    a = x;
    b = y;
}
// the same times 2^up, to the element type's largest finite value beyond that
template <typename E>
__device__ __forceinline__ void rotate(float& a, float& b, float2 w, int up) {
    turn_pair(a, b, w);
    a = saturate<E>(__builtin_ldexpf(a, up));
    b = saturate<E>(__builtin_ldexpf(b, up));
}

// A row in units of its own order. PAIRS: unit u is elements 8 u ..; those beyond rot are copied. Halves: the first `turned` units
// are eight elements and their eight partners, each other one 16 of those beyond rot, which are copied; every unit is
// computed alike (a wave holds both kinds), and the words of a copy are kept.
__host__ __device__ constexpr int turned_units(int rot) { return (rot / 2 + 7) / 8; }
__host__ __device__ constexpr int row_units(int rot, int D, bool pairs) { return pairs ? (D + 7) / 8 : turned_units(rot) + (D - rot + 15) / 16; }

struct Unit { Elems8 a, b; };
struct UnitPlace { int a, b, n_a, n_b; };   // elements, and how many of eight
// A last unit that is short begins earlier where the row goes elsewhere (twice the same bytes there): with its elements one by
// one, 8192 tokens of 40 heads, rot = 90 of 128, took 79 us, 41 so.
template <bool PAIRS>
__device__ __forceinline__ UnitPlace unit_place(int u, int rot, int D, bool in_place) {
    if constexpr (PAIRS) return {8 * u, 0, D - 8 * u, 0};
    const int half = rot / 2, turned = turned_units(rot);
    if (u < turned) {
        const int c = in_place || half < 8 ? 8 * u : min(8 * u, half - 8);
        return {c, half + c, half - c, half - c};
    }
    const int from = rot + 16 * (u - turned), c = in_place || D - rot < 16 ? from : min(from, D - 16);
    return {c, c + 8, D - c, D - c - 8};
}
template <bool PAIRS>
__device__ __forceinline__ Unit load_unit(const uint16_t* x, bool in_place, int u, int rot, int D) {
    const UnitPlace p = unit_place<PAIRS>(u, rot, D, in_place);
    Unit v{};
    v.a = load8(x + p.a, p.n_a);
    if constexpr (!PAIRS) v.b = load8(x + p.b, p.n_b);
    return v;
}
// v of load_unit, to a row that is x (in_place) or overlaps none that is read
template <typename E, bool PAIRS>
__device__ __forceinline__ void store_turned(Unit v, bool in_place, uint16_t* o, const float2* angles, int up, int u, int rot, int D) {
    const UnitPlace p = unit_place<PAIRS>(u, rot, D, in_place);
    const int half = rot / 2;
    if (in_place && (PAIRS ? 8 * u >= rot : u >= turned_units(rot))) return;
    float f[8];
    to_f32<E>(v.a, f);
    if constexpr (PAIRS) {
#pragma unroll
        for (int i = 0; i < 4; ++i) rotate<E>(f[2 * i], f[2 * i + 1], angles[min(4 * u + i, half - 1)], up);
        const Elems8 to = from_f32<E>(f);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * u + i < half) v.a.w[i] = to.w[i];
    } else {
        float g[8];
        to_f32<E>(v.b, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) rotate<E>(f[i], g[i], angles[min(p.a + i, half - 1)], up);
        if (u < turned_units(rot)) {
            v.a = from_f32<E>(f);
            v.b = from_f32<E>(g);
        }
        store8(o + p.b, v.b, p.n_b);
    }
    store8(o + p.a, v.a, p.n_a);
}

}  // namespace w4a16
