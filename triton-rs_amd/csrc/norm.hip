// Root-mean-square norm of rows with the residual's addition: h = x + r, y = h / sqrt(mean h^2 + eps) w,
// in fp32; h rounded to the element type goes back as the residual, y to the element type, or to e4m3 with a
// scale for every `group` elements: s = max(max |y| / 448, 2^-100), the fp32 quotient y / s rounded.
//
// Bound by memory: 2 bytes of x and 2 of r in, 2 of h and 2 (or 1) of y out. A row stays in the registers of
// its threads, 8 VPT elements each, so that each byte passes once; the sum of squares (and the largest |y| of a
// row) passes between them. Rows need no alignment but an element's, and no width: a thread that has fewer than eight left
// loads the row's last eight.
//
// Measured with residual, bf16: 8192 rows of 4096 48 us (5.5 TB/s), of 5003 72 (4.5), 2048 of 16384 51 (5.2); 1 row of 4096 3.1. 8-bit
// output, groups of 128: 8192 rows of 4096 45 us.
#include "elements.h"
#include "layer.h"

namespace w4a16 {

constexpr int WIDE = 0;   // TPR: a workgroup a row

// v of all threads of a row joined; 0 is neutral. Waves meet in a place of lds: 0 for the sums of squares, 1 and 2 for what is the
// largest of a row and of its result. 0 alone is used twice, with 1 between: who writes it again has passed the barrier behind
// which 1 was written, so all have read it. (1 and 2 apart, as there is no second sum of a row that is zero or not finite.)
template <int TPR, typename F>
__device__ __forceinline__ float row_all(float v, float (&lds)[3][16], int place, F f) {
    constexpr int IN_WAVE = TPR == 16 ? 16 : 64;
#pragma unroll
    for (int x = 1; x < IN_WAVE; x <<= 1) v = f(v, __shfl_xor(v, x));
    if constexpr (TPR == WIDE) {
        const int waves = blockDim.x >> 6;
        float* const at = lds[place];
        if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
        if (threadIdx.x < 16 && (int)threadIdx.x >= waves) at[threadIdx.x] = 0.f;
        __syncthreads();
        v = at[0];
#pragma unroll
        for (int x = 1; x < 16; ++x) v = f(v, at[x]);
    }
    return v;
}
// Eight elements of a row of K at its element e (zeros beyond its end, of which n = K - e are not): as one load, of the row's last
// eight where fewer are left, which `own` then moves to their places.
template <bool SHORT>
__device__ __forceinline__ Elems8 load_in(const uint16_t* row, int e, int K) {
    if constexpr (SHORT)   // K may be less than 8
        if (K < 8) return load8(row + e, K - e);
    Elems8 r = {{0, 0, 0, 0}};
    if (e < K) r = *reinterpret_cast<const Elems8*>(row + min(e, K - 8));
    return r;
}
template <bool SHORT>
__device__ __forceinline__ void own(Elems8& v, int e, int K) {
    if constexpr (SHORT)
        if (K < 8) return;
    if (e < K && e + 8 > K) v = __builtin_bit_cast(Elems8, __builtin_bit_cast(unsigned __int128, v) >> (16 * (e + 8 - K)));
}
__device__ __forceinline__ void store_in(uint16_t* row, int e, int K, const Elems8& v) {
    if (e + 8 <= K) *reinterpret_cast<Elems8*>(row + e) = v;
    else if (e < K) store8(row + e, v, K - e);
}
// The larger of two magnitudes as their bits: NaN is larger than infinity.
__device__ __forceinline__ float larger(float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }

template <typename E, bool Q8, int TPR, int VPT>
__global__ __launch_bounds__(TPR == WIDE ? 1024 : 256) void norm_kernel(NormParams p) {
    const int per_row = TPR == WIDE ? (int)blockDim.x : TPR, RPB = TPR == WIDE ? 1 : 256 / per_row;
    constexpr bool SHORT = TPR == 16 && VPT == 1;
    __shared__ float lds[3][16];
    const long long row = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * RPB + (TPR == WIDE ? 0 : threadIdx.x / per_row);
    if (row >= (long long)p.T * p.H) return;   // (a row's threads agree)
    const int t = p.H == 1 ? (int)row : (int)((unsigned)row / (unsigned)p.H), h = p.H == 1 ? 0 : (int)row - t * p.H;
    const int lane = TPR == WIDE ? threadIdx.x : threadIdx.x % per_row;
    auto at = [&](const void* base, int st, int sh) { return static_cast<const uint16_t*>(base) + (size_t)t * st + (size_t)h * sh; };
    const uint16_t *x = at(p.x, p.x_st, p.x_sh), *r = at(p.residual, p.r_st, p.r_sh), *w = static_cast<const uint16_t*>(p.weight);

    Elems8 xv[VPT], rv[VPT], wv[VPT];
    auto place = [&](int i) { return 8 * (i * per_row + lane); };
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        xv[i] = load_in<SHORT>(x, place(i), p.K);
        if (p.residual) rv[i] = load_in<SHORT>(r, place(i), p.K);
    }
    constexpr bool AHEAD = VPT <= 4;   // the weights are on their way, too (of the widest rows there are not the registers)
    if constexpr (AHEAD) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) wv[i] = load_in<SHORT>(w, place(i), p.K);
    }

    float y[VPT][8], sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        own<SHORT>(xv[i], place(i), p.K);
        to_f32<E>(xv[i], y[i]);
        if (p.residual) {
            float f[8];
            own<SHORT>(rv[i], place(i), p.K);
            to_f32<E>(rv[i], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[i][e] += f[e];
            store_in(const_cast<uint16_t*>(at(p.residual_out, p.ro_st, p.ro_sh)), place(i), p.K, from_f32<E>(y[i]));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(y[i][e], y[i][e], sum);
    }
    auto add = [](float a, float b) { return a + b; };
    sum = row_all<TPR>(sum, lds, 0, add);
    float eps = p.eps;
    // Squares that leave fp32: the row times a power of two (eps times its square), of its largest element where that
    // is large, of 2^50 at most where there is an eps that counts beside them, less where that would take eps past fp32 (which then
    // is all of the root).
    if (!(sum < 0x1p100f && sum > 0x1p-90f)) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = larger(top, __builtin_fabsf(y[i][e]));
        top = row_all<TPR>(top, lds, 1, larger);
        const int most_up = p.eps > 0.f ? min(50, max(0, 126 - (int)(__float_as_uint(p.eps) >> 24))) : 126;
        const int up = min(127 - (int)(__float_as_uint(top) >> 23), most_up);
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
            sum = row_all<TPR>(sum, lds, 0, add);
        }
    }
    const float inv = rsqrtf(sum / (float)p.K + eps);
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        float f[8];
        if constexpr (!AHEAD) wv[i] = load_in<SHORT>(w, place(i), p.K);
        own<SHORT>(wv[i], place(i), p.K);
        to_f32<E>(wv[i], f);
        if constexpr (Q8)
            if (p.group) most = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = y[i][e] * inv * f[e];
        if constexpr (!Q8) {
            store_in(const_cast<uint16_t*>(at(p.out, p.o_st, p.o_sh)), place(i), p.K, from_f32<E>(y[i]));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) most = larger(most, __builtin_fabsf(y[i][e]));
        }
    }
    if constexpr (Q8) {
        unsigned char* out = static_cast<unsigned char*>(p.out) + (size_t)t * p.o_st + (size_t)h * p.o_sh;
        if (!p.group) most = row_all<TPR>(most, lds, 2, larger);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int e0 = place(i), n = p.K - e0;
            float m = most;
            if (p.group) {
                m = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) m = larger(m, __builtin_fabsf(y[i][e]));
                for (int d = 1; d < p.group / 8; d <<= 1) m = larger(m, __shfl_xor(m, d));
            }
            float s = m / 448.f;
            s = s < 0x1p-100f ? 0x1p-100f : s;   // (NaN stays)
            // y / s in fp32 (y times the rounded 1 / s, and its rest: for s next to 2^-100 but for a unit), then to e4m3. Under an infinite
            // scale what is finite is 0.
            const float by = 1.f / s, rest = s == INFINITY ? 0.f : s;
            uint32_t q[2];
            auto over = [&](float v) {
                const float u = v * by;
                return __builtin_fmaf(__builtin_fmaf(-u, rest, v), by, u);
            };
#pragma unroll
            for (int g = 0; g < 2; ++g) q[g] = to_e4m3(over(y[i][4 * g]), over(y[i][4 * g + 1]), over(y[i][4 * g + 2]), over(y[i][4 * g + 3]));
            if (n >= 8) {
                *reinterpret_cast<Bytes8*>(out + e0) = Bytes8{{q[0], q[1]}};
            } else if (n > 0) {
#pragma unroll
                for (int e = 0; e < 7; ++e)
                    if (e < n) out[e0 + e] = (unsigned char)(q[e >> 2] >> (8 * (e & 3)));
            }
            if (p.group ? n > 0 && e0 % p.group == 0 : e0 == 0) p.scales[(size_t)row * (p.group ? p.K / p.group : 1) + (p.group ? e0 / p.group : 0)] = s;
        }
    }
}

template <typename E, bool Q8, int TPR, int VPT>
static void run(const NormParams& p, int threads, hipStream_t st) {
    const int per = TPR == WIDE ? 1 : threads / TPR;
    const long long blocks = ((long long)p.T * p.H + per - 1) / per, x = blocks < 65536 ? blocks : 65536;
    norm_kernel<E, Q8, TPR, VPT><<<dim3((unsigned)x, (unsigned)((blocks + x - 1) / x)), threads, 0, st>>>(p);
}
template <typename E, bool Q8>
static void go(const NormParams& p, hipStream_t st) {
    const int v = (p.K + 7) / 8;
    auto waves = [&](int vpt) { return (v + 64 * vpt - 1) / (64 * vpt) * 64; };
    if (v <= 16) return run<E, Q8, 16, 1>(p, 256, st);
    if (v <= 32) return run<E, Q8, 16, 2>(p, 256, st);
    if (v <= 64) return run<E, Q8, 64, 1>(p, 256, st);
    // A workgroup a row: two units a thread, so that a CU's rows are in different phases; one where rows are few (2 waves a SIMD)
    // and the time is one row's. bf16 with a residual: 8192 rows of 5120 64 us with one, 60 with two, 61 with four; 1 row of 4096
    // 3.1, 3.6, 4.3; 64 of 8192 4.0, 4.1, 4.9. To 8 bits without: 777 rows of 5003 8.4, 6.8; 300 of 8192 5.3, 4.9.
    const bool few = v <= 1024 && (long long)p.T * p.H * (waves(1) / 64) <= 2048;
    const int vpt = few ? 1 : v <= 2048 ? 2 : v <= 4096 ? 4 : 8;
    if (vpt == 1) return run<E, Q8, WIDE, 1>(p, waves(1), st);
    if (vpt == 2) return run<E, Q8, WIDE, 2>(p, waves(2), st);
    if (vpt == 4) return run<E, Q8, WIDE, 4>(p, waves(4), st);
    run<E, Q8, WIDE, 8>(p, waves(8), st);
}

hipError_t launch_norm(bool bf16, const NormParams& p, hipStream_t st) {
    if (p.group < 0) bf16 ? go<bf16_t, false>(p, st) : go<half_t, false>(p, st);
    else bf16 ? go<bf16_t, true>(p, st) : go<half_t, true>(p, st);
    return hipGetLastError();
}

}  // namespace w4a16
