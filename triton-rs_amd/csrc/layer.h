// What stands between a decoder layer's linear layers beside attention: root-mean-square norm and
// rotary positions. Launch parameters and the launchers of norm.hip and rope.hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <cmath>

namespace w4a16 {

constexpr int NORM_MAX_K = 65536;   // elements of a row: 1024 threads of 64
constexpr int64_t LAYER_MAX_ROWS = 1ll << 30;   // of a call

struct NormParams {   // rows [T, H, K], strides in elements, K contiguous
    const void *x, *residual, *weight;   // residual: null for none
    void *residual_out, *out;
    float* scales;                       // 8 bits: [T, H, K / group]
    int x_st, x_sh, r_st, r_sh, ro_st, ro_sh, o_st, o_sh;
    int T, H, K, group;                  // group: elements of a scale; -1: the result is in the element type
    float eps;
};
hipError_t launch_norm(bool bf16, const NormParams& p, hipStream_t st);

constexpr int ROPE_MAX_D = 1024;

// A rotation's factor as part 2^up, |part| <= 1: a pair of a type's largest values keeps its products within fp32, and what is
// beyond the type is infinite only where 2^up takes it there.
struct Magnitude {
    float part;
    int up;
    static Magnitude of(float m) {
        Magnitude r{m, 0};
        if (std::fabs(m) > 1.f) r.part = std::frexp(m, &r.up);
        return r;
    }
};

struct RopeRows {
    const void* x;
    void* out;
    int st, sh, o_st, o_sh, H;
};
struct RopeParams {
    RopeRows rows[2];         // queries, keys (H = 0: none)
    const int32_t* positions; // [T]
    const double* inv_freq;   // [rot / 2]
    Magnitude magnitude;
    int T, D, rot;
    bool interleaved;
};
hipError_t launch_rope(bool bf16, const RopeParams& p, hipStream_t st);

}  // namespace w4a16
