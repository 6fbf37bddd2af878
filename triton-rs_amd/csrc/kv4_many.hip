// Attention over the 4-bit cache for many columns (prompts, chunks of them): bound by the matrix and
// vector instructions. The mathematics is in kv4_attn_body.h.
//
// A workgroup of four waves takes 128 columns, 32 a wave, and walks the keys 64 at a time: each wave turns
// a block of 16 tokens into the operands n - z once for all four, in LDS and in the order in which lanes
// take them (16 bytes a lane, no bank conflicts), while the step before is computed from the other half
// of the LDS: one barrier a step. The packed words come two steps ahead into registers.
//
// Measured: 1024 queries over 32768 keys, 32 heads on 8 of D = 128, bf16, 668 us: 810 TFLOP/s, 68 % of a
// large matrix product's 1185. The matrix cores are busy in 32 % of the cycles, the vector unit in 55 %;
// two waves a SIMD is what the results leave registers for, each a chain of products, softmax and products. Steps of 32 keys with a barrier each took 861 us, logits of one half beside the
// weights of the other 754. A prompt of 2048 64 us: 512 workgroups, one to a compute unit for
// their LDS, a long tile and then a short one, 2080 keys together everywhere; at the rate above these are some 42 us, and the
// rest stands around them in either (pages, q, first blocks, the groups' join). 7 prompts of up to 1500, 16 heads of D = 64,
// 45 us. One wave a SIMD from D = 192 on: 512 queries over 8192 keys, 12 heads on 4 of 192, 102 us, 300 over 20000, 16 on 2 of
// 256, 230, a third of that product's rate.
#include "kv4_attn_body.h"

namespace w4a16 {

constexpr int MANY_STEP = 64;   // keys of a step

template <int D>
struct ManyLds {
    static constexpr int KW = D / 32, VT = D / 16;
    half8_t k[4][KW][64];      // block, word of the quarter row, lane
    half8_t v[2][VT][64];      // pair of blocks, tile of the result, lane (first block's two pairs, second's)
    float ks[64], vs[64];      // scales of the tokens, those of keys times kscale
    float above[4];            // log2_above of a block's value scales
    int live[4];               // tokens of a block that there are (0 or less: none)
};

// A lane's words of a block (of this wave): keys of token lane % 16, values of tokens 4 (lane / 16)..+3, and
// the parameters of these.
template <int D>
struct Packed {
    uint32_t k[D / 32], v[D / 32], kc;
    u32x4 vp;
};

template <int D>
__device__ __forceinline__ void load_packed(Packed<D>& t, const unsigned char* b, int lane) {
    const uint32_t ko = (lane & 15) * (D / 2) + (lane >> 4) * (D / 8), vo = 8 * D + lane * (D / 8);
    if constexpr (D % 128 == 0) {
#pragma unroll
        for (int x = 0; x < D / 128; ++x) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(at_bytes(b, ko + 16 * x)), c = *reinterpret_cast<const u32x4*>(at_bytes(b, vo + 16 * x));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                t.k[4 * x + e] = a[e];
                t.v[4 * x + e] = c[e];
            }
        }
    } else {
#pragma unroll
        for (int x = 0; x < D / 64; ++x) {
            const u32x2 a = *reinterpret_cast<const u32x2*>(at_bytes(b, ko + 8 * x)), c = *reinterpret_cast<const u32x2*>(at_bytes(b, vo + 8 * x));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                t.k[2 * x + e] = a[e];
                t.v[2 * x + e] = c[e];
            }
        }
    }
    t.kc = *reinterpret_cast<const uint32_t*>(at_bytes(b, 16 * D + (lane & 15) * 4));
    t.vp = *reinterpret_cast<const u32x4*>(at_bytes(b, 16 * D + 64 + (lane >> 4) * 16));
}

// Block `wave` of a step into LDS; its tokens [dead, live) (the others' parameters may be anything)
template <typename E, int D>
__device__ __forceinline__ void unpack(ManyLds<D>& s, Packed<D> t, int dead, int live, float kscale, uint32_t least, int wave, int lane) {
    const int col = lane & 15, kb = lane >> 4;
    t.kc = col >= dead && col < live ? t.kc : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) t.vp[i] = 4 * kb + i >= dead && 4 * kb + i < live ? t.vp[i] : 0u;
    const uint32_t zk = zeros_of(t.kc);
    const half2_t kz1 = zero1024(zk), kz16 = zero64(zk);
#pragma unroll
    for (int x = 0; x < D / 32; ++x) s.k[wave][x][lane] = key_operand(t.k[x], kz1, kz16);
    half2_t vz1[2], vz16[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        const uint32_t z = zeros_of(t.vp[2 * y], t.vp[2 * y + 1]);
        vz1[y] = zero1024(z);
        vz16[y] = zero64(z);
    }
#pragma unroll
    for (int g = 0; g < D / 64; ++g) {
        auto put = [&](auto ei) {
            constexpr int e = decltype(ei)::value;
            u32x2* dst = reinterpret_cast<u32x2*>(&s.v[wave >> 1][4 * g + e][lane]) + (wave & 1);
            *dst = u32x2{as_u32(value_pair<e>(t.v[g], vz1[0], vz16[0])), as_u32(value_pair<e>(t.v[D / 64 + g], vz1[1], vz16[1]))};
        };
        put(std::integral_constant<int, 0>{});
        put(std::integral_constant<int, 1>{});
        put(std::integral_constant<int, 2>{});
        put(std::integral_constant<int, 3>{});
    }
    if (kb == 0) s.ks[16 * wave + col] = param_scale<E>(t.kc) * kscale;
    float4_t f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = value_scale<E>(t.vp[i]);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(f[i]));
    top = kb_umax(top);
    if (col == 0) *reinterpret_cast<float4_t*>(&s.vs[16 * wave + 4 * kb]) = f;
    if (lane == 0) {
        s.above[wave] = log2_above(top, least);
        s.live[wave] = live;
    }
}

// Sequence and tile of 128 columns of this workgroup, and its chunk of the keys: those with the longest rows first, or
// (where all workgroups run at once) long and short ones by turns. p.rows: the tiles of all sequences stand in one row,
// each sequence's longest first, so that the workgroups of a prompt among single tokens lie side by side. place:
// tile and chunk, or (p.rows) chunk.
__device__ __forceinline__ bool many_tile(const Kv4AttnParams& p, int place, int& b, int& tile, int& chunk, size_t& at) {
    if (!p.rows) {
        const int z = p.splits == 1 ? place : place / p.splits;
        chunk = place - z * p.splits;
        b = blockIdx.y;
        tile = !p.pair_tiles ? p.tiles - 1 - z : z < (p.tiles + 1) / 2 ? p.tiles - 1 - z : z - (p.tiles + 1) / 2;
        at = ((size_t)tile * p.B + b) * p.Hkv + blockIdx.x;
        return true;
    }
    chunk = place;
    at = (size_t)blockIdx.y * p.Hkv + blockIdx.x;
    const int u = blockIdx.y;
    for (int base = 0, before = 0; base < p.B; base += 64) {
        const int s = base + (threadIdx.x & 63), in = min(s, p.B - 1);
        const int n = min(max(p.cu_q[in + 1], 0), p.T) - min(max(p.cu_q[in], 0), p.T);
        const int mine = s < p.B && n >= p.least_q ? (min(n, p.max_q) * p.G + 127) / 128 : 0;
        const int upto = before + wave_sums(mine);
        const uint64_t who = __ballot(u < upto);
        if (who) {
            const int l = __builtin_ctzll(who);
            b = base + l;
            tile = __builtin_amdgcn_readlane(upto, l) - 1 - u;
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

__device__ __forceinline__ bool many_item(const Kv4AttnParams& p, int place, Kv4Item& w) {
    int b, tile, chunk, lo, hi;
    w.h = blockIdx.x;
    if (!many_tile(p, place, b, tile, chunk, w.at)) return false;
    w.sequence<128, MANY_STEP>(p, b, tile * 128, lo, hi);
    const int chunks = p.splits == 1 ? 1 : max(1, (int)(((unsigned)(hi - lo) + p.chunk - 1) / (unsigned)p.chunk));
    w.take(chunk, chunks, p.chunk, lo, hi);
    w.slot = w.at * p.splits;
    return w.cols > 0 && chunk < chunks;
}

template <typename E, int D, int GROUPS>
__global__ __launch_bounds__(256 * GROUPS, kv4_many_simd_waves(D, GROUPS)) void kv4_many_kernel(Kv4AttnParams p) {
    constexpr int NT = 2, COLS = 16 * NT, STEP = MANY_STEP, ALL = STEP * GROUPS;
    typedef Kv4Cols<E, D, NT> C;
    __shared__ ManyLds<D> lds[2][GROUPS];
    __shared__ float ml[4 * COLS][2];
    Kv4Item w;
    if (!many_item(p, blockIdx.z, w)) return;
    // wave `wave` of group `group`: the group takes every GROUPS-th step of the keys
    const int lane = threadIdx.x & 63, number = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = number & 3, group = number >> 2;
    const int col = lane & 15, kb = lane >> 4;
    C a;
    a.load(p, w, w.c0 + wave * COLS, lane);

    const Kv4Pages pages(p, w, kv4_block_bytes(D));
    Packed<D> t;
    int live = 0;   // tokens of this wave's block of the step in t
    // (beyond the keys: their last block again, none of it alive)
    auto fetch = [&](int j) {
        const int blk = ((j + STEP * group) >> 4) + wave, page = pages.page(blk);
        live = pages.ok(page) ? w.k1 - 16 * blk : 0;
        load_packed<D>(t, pages.block(page, blk), lane);
    };
    const bool any = w.k0 < w.k1;
    if (any) fetch(w.k0);
    // one factor of the key scales for the workgroup's rows of q
    typename C::Sizes q = a.sizes();
    if (lane == 0 && group == 0) {   // (the groups have the same rows)
        ml[wave][0] = q.top;
        ml[wave][1] = q.top > 0.f ? q.low : INFINITY;
    }
    __syncthreads();
    q.top = fmaxf(fmaxf(ml[0][0], ml[1][0]), fmaxf(ml[2][0], ml[3][0]));
    q.low = fminf(fminf(ml[0][1], ml[1][1]), fminf(ml[2][1], ml[3][1]));
    a.start(p, q);
    __syncthreads();

    if (any) {   // (only a first step holds tokens before what its columns see)
        unpack<E, D>(lds[0][group], t, w.see_lo(p, w.n <= 1 ? 0 : w.c0 / p.G) - (w.k0 + STEP * group + 16 * wave), live, a.kscale, a.least, wave, lane);
        fetch(w.k0 + ALL);
    }
    __syncthreads();
    int buf = 0;
    for (int j = w.k0; j < w.k1; j += ALL, buf ^= 1) {
        if (j + ALL < w.k1) {
            unpack<E, D>(lds[buf ^ 1][group], t, 0, live, a.kscale, a.least, wave, lane);
            fetch(j + 2 * ALL);
        }
        const ManyLds<D>& s = lds[buf][group];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int jh = j + STEP * group + 32 * half;
            if (jh >= a.jhi || jh + 32 <= a.jlo) continue;   // none of this wave's columns sees these
            float4_t acc[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = float4_t{0.f, 0.f, 0.f, 0.f};
            float ks[2][4], vs[2][4];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const float4_t fk = *reinterpret_cast<const float4_t*>(&s.ks[32 * half + 16 * b + 4 * kb]);
                const float4_t fv = *reinterpret_cast<const float4_t*>(&s.vs[32 * half + 16 * b + 4 * kb]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    ks[b][i] = fk[i];
                    vs[b][i] = fv[i];
                }
            }
            // operands from LDS all at once, ahead of what takes them: one wait instead of eight
            half8_t kf[2][C::KW], vf[C::VT];
            const int live0 = s.live[2 * half], live1 = s.live[2 * half + 1];
            const float above0 = s.above[2 * half], above1 = s.above[2 * half + 1];
#pragma unroll
            for (int x = 0; x < C::KW; ++x)
#pragma unroll
                for (int b = 0; b < 2; ++b) kf[b][x] = s.k[2 * half + b][x][lane];
            __builtin_amdgcn_sched_barrier(0);
            const int bad = __builtin_amdgcn_readfirstlane((live0 <= 0 ? 1 : 0) | (live1 <= 0 ? 2 : 0));
            const bool whole = jh >= a.all_lo && jh + 32 <= a.all_hi && jh + 32 <= a.jhi && !bad;
            const float above = fmaxf(above0, above1);
#pragma unroll
            for (int x = 0; x < C::KW; ++x)
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int n = 0; n < NT; ++n) acc[n][b] = mfma16x16x32(kf[b][x], a.qf[n][x], acc[n][b]);
            a.uncommon(acc, ks, vs, above, whole, jh, a.jhi, bad, kb);
            float x[NT][2][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) a.logits(n, x[n], acc[n], ks, vs, above, whole, jh, a.jhi, bad, kb);
#pragma unroll
            for (int x = 0; x < C::VT; ++x) vf[x] = s.v[half][x][lane];
            __builtin_amdgcn_sched_barrier(0);
            half8_t pw[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) pw[n] = a.weights(n, x[n], vs);
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
    const Kv4Sink<E, D> sink(p, w);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if (group) break;
        const int c = 16 * n + col;
        const float inv = over_sum<E>(a.l[n]);
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

// Joins the chunks of one tile: an eighth of its values a workgroup. (The last of the chunks' own workgroups took longer:
// 64 queries over 4096 keys, 32 heads of D = 128, 8 chunks, 40.1 us, so 30; two chunks of 400 over 2000 40.2, 39.3.)
constexpr int MANY_PARTS = 8;
template <typename E, int D>
__global__ __launch_bounds__(256) void kv4_many_join_kernel(Kv4AttnParams p) {
    __shared__ float ml[128][2];
    Kv4Item w;
    const int part = blockIdx.z % MANY_PARTS;
    if (!many_item(p, blockIdx.z / MANY_PARTS * p.splits, w) || w.chunks == 1) return;   // (its results are in place)
    const Kv4Sink<E, D> sink(p, w);
    sink.template join_lanes<MANY_PARTS>(min(128, w.cols), &ml[0][0], part);
}

template <typename E, int D>
static void go(const Kv4AttnShape& s, const Kv4AttnParams& p, hipStream_t st) {
    const dim3 grid = s.rows ? dim3(p.Hkv, s.rows, s.splits) : dim3(p.Hkv, p.B, s.tiles * s.splits);
    auto join = [&] {
        const dim3 parts(grid.x, grid.y, (s.rows ? 1 : s.tiles) * MANY_PARTS);
        if (s.splits > 1) kv4_many_join_kernel<E, D><<<parts, 256, 0, st>>>(p);
    };
    if constexpr (D <= 128)
        if (s.groups == 2) {
            kv4_many_kernel<E, D, 2><<<grid, 512, 0, st>>>(p);
            join();
            return;
        }
    kv4_many_kernel<E, D, 1><<<grid, 256, 0, st>>>(p);
    join();
}

hipError_t launch_kv4_many(bool bf16, int D, const Kv4AttnParams& p, const Kv4AttnShape& s, hipStream_t st) {
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
