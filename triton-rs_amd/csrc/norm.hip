// Root-mean-square norm of rows with the residual's addition: h = x + r, y = h / sqrt(mean h^2 + eps) w,
// in fp32; h rounded to the element type goes back as the residual, y to the element type, or to e4m3 with a
// scale for every `group` elements: s = max(max |y| / 448, 2^-100), y / s rounded.
//
// Bound by memory: 2 bytes of x and 2 of r in, 2 of h and 2 (or 1) of y out. A row stays in the registers of
// TPR threads, 8 VPT elements each, so that each byte passes once; the sum of squares (and the largest |y| of a
// row) passes between them. Rows need no alignment but an element's, and no width: the last thread takes what
// is left of eight one by one.
#include "elements.h"
#include "layer.h"

namespace w4a16 {

template <int TPR, typename F>
__device__ __forceinline__ float row_all(float v, float* lds, F f) {
    constexpr int IN_WAVE = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int x = 1; x < IN_WAVE; x <<= 1) v = f(v, __shfl_xor(v, x));
    if constexpr (TPR > 64) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();   // (an earlier sum has been read)
        if ((threadIdx.x & 63) == 0) lds[wave] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int x = 1; x < TPR / 64; ++x) v = f(v, lds[x]);
    }
    return v;
}
// The larger of two magnitudes as their bits: NaN is larger than infinity.
__device__ __forceinline__ float larger(float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }

template <typename E, bool Q8, int TPR, int VPT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_kernel(NormParams p) {
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
    __shared__ float lds[TPR > 64 ? TPR / 64 : 1];
    const long long row = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * RPB + threadIdx.x / TPR;
    if (row >= (long long)p.T * p.H) return;   // (a row's threads agree)
    const int t = p.H == 1 ? (int)row : (int)((unsigned)row / (unsigned)p.H), h = p.H == 1 ? 0 : (int)row - t * p.H;
    const int lane = threadIdx.x % TPR;
    auto at = [&](const void* base, int st, int sh) { return static_cast<const uint16_t*>(base) + (size_t)t * st + (size_t)h * sh; };
    const uint16_t *x = at(p.x, p.x_st, p.x_sh), *r = at(p.residual, p.r_st, p.r_sh), *w = static_cast<const uint16_t*>(p.weight);

    Elems8 xv[VPT], rv[VPT], wv[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int e = 8 * (i * TPR + lane);
        xv[i] = load8(x + e, p.K - e);
        if (p.residual) rv[i] = load8(r + e, p.K - e);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) wv[i] = load8(w + 8 * (i * TPR + lane), p.K - 8 * (i * TPR + lane));

    float y[VPT][8], sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        to_f32<E>(xv[i], y[i]);
        if (p.residual) {
            float f[8];
            to_f32<E>(rv[i], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[i][e] += f[e];
            store8(const_cast<uint16_t*>(at(p.residual_out, p.ro_st, p.ro_sh)) + 8 * (i * TPR + lane), from_f32<E>(y[i]), p.K - 8 * (i * TPR + lane));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(y[i][e], y[i][e], sum);
    }
    auto add = [](float a, float b) { return a + b; };
    sum = row_all<TPR>(sum, lds, add);
    float eps = p.eps;
    // Squares that leave fp32: the row times a power of two (eps times its square), of its largest element where that
    // is large, of 2^50 at most where there is an eps that counts beside them.
    if (!(sum < 0x1p100f && sum > 0x1p-90f)) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = larger(top, __builtin_fabsf(y[i][e]));
        top = row_all<TPR>(top, lds, larger);
        const int up = min(127 - (int)(__float_as_uint(top) >> 23), p.eps > 0.f ? 50 : 126);
        if (top > 0.f && top < INFINITY) {
            eps = __builtin_ldexpf(eps, 2 * up);
            sum = 0.f;
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    y[i][e] = __builtin_ldexpf(y[i][e], up);
                    sum = __builtin_fmaf(y[i][e], y[i][e], sum);
                }
            sum = row_all<TPR>(sum, lds, add);
        }
    }
    const float inv = rsqrtf(sum / (float)p.K + eps);
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        float f[8];
        to_f32<E>(wv[i], f);
        if constexpr (Q8)
            if (p.group) most = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = y[i][e] * inv * f[e];
        if constexpr (!Q8) {
            store8(const_cast<uint16_t*>(at(p.out, p.o_st, p.o_sh)) + 8 * (i * TPR + lane), from_f32<E>(y[i]), p.K - 8 * (i * TPR + lane));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) most = larger(most, __builtin_fabsf(y[i][e]));
        }
    }
    if constexpr (Q8) {
        unsigned char* out = static_cast<unsigned char*>(p.out) + (size_t)t * p.o_st + (size_t)h * p.o_sh;
        if (!p.group) most = row_all<TPR>(most, lds, larger);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int e0 = 8 * (i * TPR + lane), n = p.K - e0;
            float m = most;
            if (p.group) {
                m = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) m = larger(m, __builtin_fabsf(y[i][e]));
                for (int d = 1; d < p.group / 8; d <<= 1) m = larger(m, __shfl_xor(m, d));
            }
            float s = m / 448.f;
            s = s < 0x1p-100f ? 0x1p-100f : s;   // (NaN stays)
            const float by = 1.f / s;
            uint32_t q[2];
#pragma unroll
            for (int g = 0; g < 2; ++g) q[g] = to_e4m3(y[i][4 * g] * by, y[i][4 * g + 1] * by, y[i][4 * g + 2] * by, y[i][4 * g + 3] * by);
            if (n >= 8) {
                *reinterpret_cast<Bytes8*>(out + e0) = Bytes8{{q[0], q[1]}};
            } else {
#pragma unroll
                for (int e = 0; e < 7; ++e)
                    if (e < n) out[e0 + e] = (unsigned char)(q[e >> 2] >> (8 * (e & 3)));
            }
            if (p.group ? n > 0 && e0 % p.group == 0 : e0 == 0) p.scales[(size_t)row * (p.group ? p.K / p.group : 1) + (p.group ? e0 / p.group : 0)] = s;
        }
    }
}

template <typename E, bool Q8, int TPR, int VPT>
static void run(const NormParams& p, hipStream_t st) {
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
    const long long blocks = ((long long)p.T * p.H + RPB - 1) / RPB, x = blocks < 65536 ? blocks : 65536;
    norm_kernel<E, Q8, TPR, VPT><<<dim3((unsigned)x, (unsigned)((blocks + x - 1) / x)), TPR < 256 ? 256 : TPR, 0, st>>>(p);
}
template <typename E, bool Q8>
static void go(const NormParams& p, hipStream_t st) {
    const int v = (p.K + 7) / 8;
    if (v <= 16) return run<E, Q8, 16, 1>(p, st);
    if (v <= 32) return run<E, Q8, 16, 2>(p, st);
    if (v <= 64) return run<E, Q8, 64, 1>(p, st);
    if (v <= 128) return run<E, Q8, 64, 2>(p, st);
    if (v <= 256) return run<E, Q8, 256, 1>(p, st);
    if (v <= 512) return run<E, Q8, 256, 2>(p, st);
    if (v <= 1024) return run<E, Q8, 256, 4>(p, st);
    if (v <= 2048) return run<E, Q8, 256, 8>(p, st);
    if (v <= 4096) return run<E, Q8, 1024, 4>(p, st);
    run<E, Q8, 1024, 8>(p, st);
}

hipError_t launch_norm(bool bf16, const NormParams& p, hipStream_t st) {
    if (p.group < 0) bf16 ? go<bf16_t, false>(p, st) : go<half_t, false>(p, st);
    else bf16 ? go<bf16_t, true>(p, st) : go<half_t, true>(p, st);
    return hipGetLastError();
}

}  // namespace w4a16
