// Attention over the 8-bit cache for many columns (prompts, chunks of them): bound by the matrix and
// vector instructions. The mathematics is in kv8_attn_body.h.
//
// A workgroup of four waves takes 128 columns, 32 a wave, and walks the keys 64 at a time: each wave turns
// a block of 16 tokens into operands once for all four, in LDS and in the order in which lanes take them (16
// bytes a lane, no bank conflicts), while the step before is computed from the other half of the LDS: one
// barrier a step. The bytes come two steps ahead into registers.
#include "kv8_attn_body.h"
#include "kv_many.h"

namespace w4a16 {

template <typename E, int D>
struct ManyLds {
    static constexpr int KW = D / 32, VT = D / 16;
    typename vec8<E>::type k[4][KW][64];   // block, operand of a row, lane
    half8_t v[2][VT][64];                  // pair of blocks, tile of the result, lane (first block's tokens, second's)
    Kv8Scale scale[4];
    int live[4];                           // tokens of a block that there are (0 or less: none)
};

// A block (of this wave) as this lane takes it.
template <int D>
struct Packed {
    u32x4 k[D / 64], v[D / 64];
    u32x3 tail;
};

// Block `wave` of a step into LDS; its tokens [dead, live) (the others' bytes may be anything)
template <typename E, int D>
__device__ __forceinline__ void unpack(ManyLds<E, D>& s, const Packed<D>& t, int dead, int live, float factor, int wave, int lane) {
    const uint32_t mask = dead <= 0 && live >= 16 ? ~0u : token_bytes(dead, live, lane >> 4);
#pragma unroll
    for (int g = 0; g < D / 64; ++g) {
#pragma unroll
        for (int h = 0; h < 2; ++h) s.k[wave][2 * g + h][lane] = operand8<E>(t.k[g][2 * h], t.k[g][2 * h + 1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t w = t.v[g][e] & mask;
            *(reinterpret_cast<u32x2*>(&s.v[wave >> 1][4 * g + e][lane]) + (wave & 1)) = u32x2{from_e4m3<half_t, false>(w), from_e4m3<half_t, true>(w)};
        }
    }
    if (lane == 0) {
        s.scale[wave] = Kv8Scale::of(t.tail, factor, live > 0 && dead < 16);
        s.live[wave] = live;
    }
}

template <typename E, int D, int GROUPS>
__global__ __launch_bounds__(256 * GROUPS, kv8_many_simd_waves(D, GROUPS)) void kv8_many_kernel(KvAttnParams p) {
    constexpr int NT = 2, COLS = 16 * NT, STEP = MANY_STEP, ALL = STEP * GROUPS;
    typedef Kv8Cols<E, D, NT> C;
    __shared__ ManyLds<E, D> lds[2][GROUPS];
    KvItem w;
    if (!many_item(p, blockIdx.z, w)) return;
    // wave `wave` of group `group`: the group takes every GROUPS-th step of the keys
    const int lane = threadIdx.x & 63, number = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = number & 3, group = number >> 2;
    const int col = lane & 15, kb = lane >> 4;
    C a;
    a.load(p, w, w.c0 + wave * COLS, lane);

    const KvPages pages(p, w, kv8_block_bytes(D));
    Packed<D> t;
    int live = 0;   // tokens of this wave's block of the step in t
    // (beyond the keys: their last block again, none of it alive; the page of the step after it ahead of its use)
    int page = 0;
    auto block_of = [&](int j) { return ((j + STEP * group) >> 4) + wave; };
    auto fetch = [&](int j) {
        const int blk = block_of(j);
        live = pages.ok(page) ? w.k1 - 16 * blk : 0;
        const unsigned char* b = pages.block(page, blk);
#pragma unroll
        for (int g = 0; g < D / 64; ++g) t.k[g] = *reinterpret_cast<const u32x4*>(at_bytes(b, 1024 * g + 16 * lane));
#pragma unroll
        for (int g = 0; g < D / 64; ++g) t.v[g] = *reinterpret_cast<const u32x4*>(at_bytes(b, 16 * D + 1024 * g + 16 * lane));
        t.tail = block_tail(b, D);
        page = pages.page(block_of(j + ALL));
    };
    const bool any = w.k0 < w.k1;
    if (any) {
        page = pages.page(block_of(w.k0));
        fetch(w.k0);
    }
    a.start();
    if (any) {   // (only a first step holds tokens before what its columns see)
        unpack<E, D>(lds[0][group], t, w.see_lo(p, w.n <= 1 ? 0 : w.c0 / p.G) - (w.k0 + STEP * group + 16 * wave), live, p.scale_log2, wave, lane);
        fetch(w.k0 + ALL);
    }
    __syncthreads();
    int buf = 0;
    for (int j = w.k0; j < w.k1; j += ALL, buf ^= 1) {
        if (j + ALL < w.k1) {
            unpack<E, D>(lds[buf ^ 1][group], t, 0, live, p.scale_log2, wave, lane);
            fetch(j + 2 * ALL);
        }
        const ManyLds<E, D>& s = lds[buf][group];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int jh = j + STEP * group + 32 * half;
            if (jh >= a.jhi || jh + 32 <= a.jlo) continue;   // none of this wave's columns sees these
            float4_t acc[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = float4_t{0.f, 0.f, 0.f, 0.f};
            // operands from LDS all at once, ahead of what takes them: one wait instead of eight
            typename C::vec_t kf[2][C::KW];
            half8_t vf[C::VT];
            Kv8Scale sc[2] = {s.scale[2 * half], s.scale[2 * half + 1]};
            const int live0 = s.live[2 * half], live1 = s.live[2 * half + 1];
#pragma unroll
            for (int x = 0; x < C::KW; ++x)
#pragma unroll
                for (int b = 0; b < 2; ++b) kf[b][x] = s.k[2 * half + b][x][lane];
            __builtin_amdgcn_sched_barrier(0);
            const int bad = __builtin_amdgcn_readfirstlane((live0 <= 0 ? 1 : 0) | (live1 <= 0 ? 2 : 0));
            sc[0].nan = __builtin_amdgcn_readfirstlane(sc[0].nan);
            sc[1].nan = __builtin_amdgcn_readfirstlane(sc[1].nan);
            const bool whole = jh >= a.all_lo && jh + 32 <= a.all_hi && jh + 32 <= a.jhi && !bad && !(sc[0].nan | sc[1].nan);
#pragma unroll
            for (int x = 0; x < C::KW; ++x)
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int n = 0; n < NT; ++n) acc[n][b] = mfma16x16x32(kf[b][x], a.qf[n][x], acc[n][b]);
            float x[NT][2][4], back[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) a.logits(n, x[n], back[n], acc[n], sc, whole, jh, a.jhi, bad, kb);
#pragma unroll
            for (int x = 0; x < C::VT; ++x) vf[x] = s.v[half][x][lane];
            __builtin_amdgcn_sched_barrier(0);
                half8_t pw[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) pw[n] = a.weights(n, x[n], back[n]);
#pragma unroll
            for (int x = 0; x < C::VT; ++x)
#pragma unroll
                for (int n = 0; n < NT; ++n) a.o[n][x] = mfma16x16x32(vf[x], pw[n], a.o[n][x]);
        }
        __syncthreads();
    }
    a.finish();

    if constexpr (GROUPS == 2) {   // the second group's share of the keys to the first
        float4_t* const o = reinterpret_cast<float4_t*>(&lds[0][0]) + wave * (NT * C::VT) * 64;
        float* const mls = reinterpret_cast<float*>(reinterpret_cast<float4_t*>(&lds[0][0]) + 4 * (NT * C::VT) * 64) + wave * NT * 128;
        static_assert(4 * NT * C::VT * 64 * 16 + 4 * NT * 128 * 4 <= sizeof(lds), "results of four waves fit");
        if (group) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                mls[128 * n + lane] = a.m[n];
                mls[128 * n + 64 + lane] = a.l[n];
#pragma unroll
                for (int x = 0; x < C::VT; ++x) o[(n * C::VT + x) * 64 + lane] = a.o[n][x];
            }
        }
        __syncthreads();
        if (group == 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float m1 = mls[128 * n + lane], mm = fmaxf(a.m[n], m1);
                const float h0 = half_fall(a.m[n], mm), h1 = half_fall(m1, mm), f0 = h0 * h0, f1 = h1 * h1;
                a.m[n] = mm;
                a.l[n] = a.l[n] * h0 * h0 + mls[128 * n + 64 + lane] * h1 * h1;
#pragma unroll
                for (int x = 0; x < C::VT; ++x) a.o[n][x] = a.o[n][x] * f0 + o[(n * C::VT + x) * 64 + lane] * f1;
            }
        }
    }
    const KvSink<E, D, 0> sink(p, w);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if (group) break;
        const int c = 16 * n + col;
        const float inv = over_sum<0>(a.l[n]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int x = 0; x < C::VT; x += 4) {
                const float4_t v = {a.o[n][x][i], a.o[n][x + 1][i], a.o[n][x + 2][i], a.o[n][x + 3][i]};
                // (chunks of partial results as they lie: 1 KiB a store and wave)
                if (w.chunks > 1) {
                    st_partial4<SCOPE_DEVICE>(sink.part + 4 * sink.lane_quad(wave, n, i, x, lane), v);
                } else if (c < a.n) {
                    if constexpr (C::VT % 8 == 0) {   // 16 bytes a store
                        if (x % 8 == 4) sink.out8(a.c + c, (4 * kb + i) * C::VT + x - 4, float4_t{a.o[n][x - 4][i], a.o[n][x - 3][i], a.o[n][x - 2][i], a.o[n][x - 1][i]}, v, inv);
                    } else {
                        sink.out(a.c + c, (4 * kb + i) * C::VT + x, v, inv);
                    }
                }
            }
        if (kb == 0 && c < a.n) sink.put_ml(a.c + c, a.m[n], a.l[n]);
    }
}

template <typename E, int D>
__global__ __launch_bounds__(256) void kv8_many_join_kernel(KvAttnParams p) {
    __shared__ float ml[128][2];
    many_join<E, D, 0>(p, &ml[0][0]);
}

template <typename E, int D>
static void go(const KvAttnShape& s, const KvAttnParams& p, hipStream_t st) {
    const dim3 grid = s.rows ? dim3(p.Hkv, s.rows, s.splits) : dim3(p.Hkv, p.B, s.tiles * s.splits);
    auto join = [&] {
        const dim3 parts(grid.x, grid.y, (s.rows ? 1 : s.tiles) * MANY_PARTS);
        if (s.splits > 1) kv8_many_join_kernel<E, D><<<parts, 256, 0, st>>>(p);
    };
    if constexpr (D <= 128)
        if (s.groups == 2) {
            kv8_many_kernel<E, D, 2><<<grid, 512, 0, st>>>(p);
            join();
            return;
        }
    kv8_many_kernel<E, D, 1><<<grid, 256, 0, st>>>(p);
    join();
}

hipError_t launch_kv8_many(bool bf16, int D, const KvAttnParams& p, const KvAttnShape& s, hipStream_t st) {
    switch (D) {
        case 64: bf16 ? go<bf16_t, 64>(s, p, st) : go<half_t, 64>(s, p, st); break;
        case 128: bf16 ? go<bf16_t, 128>(s, p, st) : go<half_t, 128>(s, p, st); break;
        case 192: bf16 ? go<bf16_t, 192>(s, p, st) : go<half_t, 192>(s, p, st); break;
        case 256: bf16 ? go<bf16_t, 256>(s, p, st) : go<half_t, 256>(s, p, st); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace w4a16
