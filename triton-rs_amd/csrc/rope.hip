// Rotary positions: pair (a, b) of a row, dimensions (i, i + rot / 2) or (2 i, 2 i + 1), at position n becomes
// m (a cos w - b sin w, a sin w + b cos w), w = n f_i, in fp32, rounded once.
//
// An angle is taken modulo a whole turn in fp64 (a position of 10^6 in fp32 would be off by 0.06 rad); its
// sine and cosine (rotate.h) are computed once a token for all heads, in LDS. The two products of a
// result are rounded before their difference or sum, so that every kernel that rotates gives the same bits.
// Bound by memory: a row in, a row out. 8192 tokens, 40 heads of D = 128, 168 MB: 37 us (4.5 TB/s), rot = 64, 90 or 96 of it
// 40, 41 and 37; 16 tokens 3.7.
#include "elements.h"
#include "layer.h"
#include "rotate.h"

namespace w4a16 {

constexpr int ROPE_TOKENS = 2;   // of a workgroup, at most
struct RowPlace { const uint16_t* x; uint16_t* o; };

template <typename E, bool PAIRS>
__global__ __launch_bounds__(256) void rope_kernel(RopeParams p, int tokens) {
    extern __shared__ float2 turn[];   // [tokens][rot / 2]
    const int half = p.rot / 2, t0 = (int)(blockIdx.y * gridDim.x + blockIdx.x) * tokens, live = min(tokens, p.T - t0);
    if (live <= 0) return;
    const int units = row_units(p.rot, p.D, PAIRS);
    static_assert(ROPE_MAX_D / 8 + 1 <= 256, "a row's units are threads of one workgroup");
    const int rows = 256 / units, heads = p.rows[0].H + p.rows[1].H, all = live * heads;
    const int mine = threadIdx.x / units, u = threadIdx.x - mine * units;
    auto row = [&](int r, int& t) {   // row r of the workgroup
        t = r / heads;
        const int hh = r - t * heads;
        const bool second = hh >= p.rows[0].H;
        const RopeRows& w = p.rows[second];
        const int h = second ? hh - p.rows[0].H : hh;
        return RowPlace{static_cast<const uint16_t*>(w.x) + (size_t)(t0 + t) * w.st + (size_t)h * w.sh,
                        static_cast<uint16_t*>(w.out) + (size_t)(t0 + t) * w.o_st + (size_t)h * w.o_sh};
    };
    for (int r0 = 0; r0 < all; r0 += rows) {
        const int r = r0 + mine;
        const bool some = mine < rows && r < all;
        Unit v{};
        int t = 0;
        RowPlace at{};
        if (some) {
            at = row(r, t);
            v = load_unit<PAIRS>(at.x, at.x == at.o, u, p.rot, p.D);
        }
        if (r0 == 0) {   // while the first rows are on their way
            for (int i = threadIdx.x; i < live * half; i += 256) {
                const int t = i / half;
                turn[i] = angle(p.positions[t0 + t], p.inv_freq[i - t * half], p.magnitude.part);
            }
            __syncthreads();
        }
        if (some) store_turned<E, PAIRS>(v, at.x == at.o, at.o, turn + t * half, p.magnitude.up, u, p.rot, p.D);
    }
}

template <typename E>
static void go(const RopeParams& p, hipStream_t st) {
    // Two tokens a workgroup where all of them are more than are resident at once; with one its angles and barrier count (8192
    // tokens, 40 heads of D = 64 20 us and 18), with four a CU's workgroups all wait at once (40 heads of 128, pairs: 38 and 43 us).
    const int tokens = p.T >= 2048 ? ROPE_TOKENS : 1;
    const unsigned blocks = ((unsigned)p.T + tokens - 1) / tokens, x = blocks < 65536 ? blocks : 65536;   // (a launch's threads along x are 32-bit)
    const dim3 grid(x, (blocks + x - 1) / x);
    const size_t lds = sizeof(float2) * tokens * (p.rot / 2);
    if (p.interleaved) rope_kernel<E, true><<<grid, 256, lds, st>>>(p, tokens);
    else rope_kernel<E, false><<<grid, 256, lds, st>>>(p, tokens);
}

hipError_t launch_rope(bool bf16, const RopeParams& p, hipStream_t st) {
    bf16 ? go<bf16_t>(p, st) : go<half_t>(p, st);
    return hipGetLastError();
}

}  // namespace w4a16
