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

}  // namespace w4a16
