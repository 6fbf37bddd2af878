// Rotary positions: pair (a, b) of a row, dimensions (i, i + rot / 2) or (2 i, 2 i + 1), at position n becomes
// m (a cos w - b sin w, a sin w + b cos w), w = n f_i, in fp32, rounded once.
//
// An angle is taken modulo a whole turn in fp64 (a position of 10^6 in fp32 would be off by 0.06 rad) and its
// sine and cosine, fp64 rounded to fp32, are computed once a token for all heads, in LDS. The two products of a
// result are rounded before their difference or sum, so that every kernel that rotates gives the same bits.
// Bound by memory: a row in, a row out.
#include "elements.h"
#include "layer.h"
#include "rotate.h"

namespace w4a16 {

template <typename E, bool PAIRS>
__global__ __launch_bounds__(256) void rope_kernel(RopeParams p, int tokens) {
    extern __shared__ float2 turn[];   // [tokens][rot / 2]
    const int half = p.rot / 2, t0 = blockIdx.x * tokens, live = min(tokens, p.T - t0);
    for (int i = threadIdx.x; i < live * half; i += 256) {
        const int t = i / half;
        turn[i] = angle(p.positions[t0 + t], p.inv_freq[i - t * half], p.magnitude);
    }
    __syncthreads();
    const int turned = turned_units(p.rot, PAIRS), units = row_units(p.rot, p.D, PAIRS);
    static_assert(ROPE_MAX_D / 8 + 1 <= 256, "a row's units are threads of one workgroup");
    const int rows = 256 / units, heads = p.rows[0].H + p.rows[1].H;
    const int mine = threadIdx.x / units, u = threadIdx.x - mine * units;
    if (mine >= rows) return;
    for (int r = mine; r < live * heads; r += rows) {
        const int t = r / heads, hh = r - t * heads;
        const RopeRows& w = p.rows[hh >= p.rows[0].H];
        const int h = hh >= p.rows[0].H ? hh - p.rows[0].H : hh;
        turn_unit<E, PAIRS>(static_cast<const uint16_t*>(w.x) + (size_t)(t0 + t) * w.st + (size_t)h * w.sh,
                            static_cast<uint16_t*>(w.out) + (size_t)(t0 + t) * w.o_st + (size_t)h * w.o_sh, turn + t * half, u, turned, p.rot, p.D);
    }
}

template <typename E>
static void go(const RopeParams& p, hipStream_t st) {
    const int tokens = p.T >= 4096 ? 4 : 1;
    const dim3 grid((unsigned)((p.T + tokens - 1) / tokens));
    const size_t lds = sizeof(float2) * tokens * (p.rot / 2);
    if (p.interleaved) rope_kernel<E, true><<<grid, 256, lds, st>>>(p, tokens);
    else rope_kernel<E, false><<<grid, 256, lds, st>>>(p, tokens);
}

hipError_t launch_rope(bool bf16, const RopeParams& p, hipStream_t st) {
    bf16 ? go<bf16_t>(p, st) : go<half_t>(p, st);
    return hipGetLastError();
}

}  // namespace w4a16
