// Attention over the 8-bit cache for few columns (at most 64 of a key/value head: single tokens, drafts):
// bound by the cache's bytes. The mathematics is in kv8_attn_body.h.
//
// The waves of a workgroup share their columns' keys, every second or fourth step of 32 each, and
// join through LDS. A block lies in memory in the order in which lanes take their operands, so a wave loads its
// steps into registers, 1 KiB an instruction, one step ahead of the one that it computes. The keys of a
// sequence are split into chunks only as far as it takes to fill the device.
#include "kv8_attn_body.h"
#include "kv_few.h"

namespace w4a16 {

template <typename E, int D, int NT>
__global__ __launch_bounds__(256, kv8_few_occupancy(D, NT)) void kv8_few_kernel(KvAttnParams p) {
    typedef Kv8Cols<E, D, NT> C;
    constexpr int COLS = 16 * NT, ROW = D + 4;   // LDS row of a column's result
    __shared__ __align__(16) float red[4][16 * ROW];
    static_assert(4096 + 2048 <= sizeof(red), "what joins chunks fits");
    __shared__ float ml[4][COLS][2];
    __shared__ int last;
    __shared__ FewFind find;
    KvItem w;
    if (!few_item<2 * COLS>(p, blockIdx.y, blockIdx.z, false, w, find)) return;
    // one group of columns, its keys over four waves, or two over two
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kshift = w.cols <= COLS ? 2 : 1, kspl = 1 << kshift, g0 = wave & ~(kspl - 1);
    const int col = lane & 15, kb = lane >> 4;

    C a;
    a.load(p, w, w.c0 + (wave >> kshift) * COLS, lane);
    const int stride = STEP << kshift, beg = __builtin_amdgcn_readfirstlane((a.jlo & ~(STEP - 1)) + STEP * (wave & (kspl - 1))), end = __builtin_amdgcn_readfirstlane(a.jhi);
    const KvPages pages(p, w, kv8_block_bytes(D));
    // One step of keys and one of values in registers: the next step's keys are loaded over this one's as soon as the first product
    // has taken them, its values behind the second. (Steps beyond the last load its last block again; none is computed.)
    u32x4 k[2][D / 64], v[2][D / 64];
    u32x3 tail[2];
    int bad = 0;   // bit b: block b of the step lies in no page
    const unsigned char* block[2];
    auto locate = [&](int at, int pa, int pb) {
        block[0] = pages.block(pa, at >> 4);
        block[1] = pages.block(pb, (at >> 4) + 1);
    };
    auto load_keys = [&] {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int g = 0; g < D / 64; ++g) k[b][g] = *reinterpret_cast<const u32x4*>(at_bytes(block[b], 1024 * g + 16 * lane));
    };
    auto load_values = [&] {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int g = 0; g < D / 64; ++g) v[b][g] = *reinterpret_cast<const u32x4*>(at_bytes(block[b], 16 * D + 1024 * g + 16 * lane));
    };
    auto load_tails = [&] {
#pragma unroll
        for (int b = 0; b < 2; ++b) tail[b] = block_tail(block[b], D);
    };
    a.start();
    if (beg < end) {
        auto page = [&](int at, int b) { return pages.page((at >> 4) + b); };
        int pa = page(beg, 0), pb = page(beg, 1);
        locate(beg, pa, pb);
        load_keys();
        load_tails();
        load_values();
        bad = (pages.ok(pa) ? 0 : 1) | (pages.ok(pb) ? 0 : 2);
        pa = page(beg + stride, 0);
        pb = page(beg + stride, 1);
        for (int j = beg; j < end; j += stride) {
            float4_t acc[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < C::KW; ++x)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const auto f = operand8<E>(k[b][x >> 1][2 * (x & 1)], k[b][x >> 1][2 * (x & 1) + 1]);
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[t][b] = mfma16x16x32(f, a.qf[t][x], acc[t][b]);
                }
            locate(j + stride, pa, pb);
            load_keys();
            __builtin_amdgcn_sched_barrier(0);
            const Kv8Scale sc[2] = {Kv8Scale::of(tail[0], p.scale_log2, !(bad & 1) && j + 16 > a.jlo),
                                    Kv8Scale::of(tail[1], p.scale_log2, !(bad & 2) && j + 16 < end && j + 32 > a.jlo)};
            const bool whole = j >= a.all_lo && j + STEP <= a.all_hi && j + STEP <= end && !bad && !__builtin_amdgcn_readfirstlane(sc[0].nan | sc[1].nan);
            // bytes of tokens that no column sees may be anything
            uint32_t mask[2] = {~0u, ~0u};
            if (!whole)
#pragma unroll
                for (int b = 0; b < 2; ++b) mask[b] = token_bytes(a.jlo - j - 16 * b, (bad >> b) & 1 ? 0 : end - j - 16 * b, kb);
            half8_t pw[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float x[2][4], back[2];
                a.logits(t, x, back, acc[t], sc, whole, j, end, bad, kb);
                pw[t] = a.weights(t, x, back);
            }
            load_tails();
#pragma unroll
            for (int g = 0; g < D / 64; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const half8_t f = operand8<half_t>(v[0][g][e] & mask[0], v[1][g][e] & mask[1]);
#pragma unroll
                    for (int t = 0; t < NT; ++t) a.o[t][4 * g + e] = mfma16x16x32(f, pw[t], a.o[t][4 * g + e]);
                }
            load_values();
            bad = __builtin_amdgcn_readfirstlane((pages.ok(pa) ? 0 : 1) | (pages.ok(pb) ? 0 : 2));
            pa = page(j + 2 * stride, 0);
            pb = page(j + 2 * stride, 1);
        }
    }
    a.finish();

    // the waves of a group join their shares of the keys
    const KvSink<E, D, 0> sink(p, w);
#pragma unroll
    for (int t = 0; t < NT; ++t)
        if (kb == 0) {
            ml[wave][16 * t + col][0] = a.m[t];
            ml[wave][16 * t + col][1] = a.l[t];
        }
    __syncthreads();
    const int u = threadIdx.x & (64 * kspl - 1);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float top = ml[g0][16 * t + col][0];
        for (int x = 1; x < kspl; ++x) top = fmaxf(top, ml[g0 + x][16 * t + col][0]);
        const float f = half_fall(a.m[t], top);
        if (t) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int x = 0; x < C::VT; x += 4)
                *reinterpret_cast<float4_t*>(red[wave] + col * ROW + (4 * kb + i) * C::VT + x) =
                    float4_t{a.o[t][x][i], a.o[t][x + 1][i], a.o[t][x + 2][i], a.o[t][x + 3][i]} * f * f;
        __syncthreads();
        const int live = min(16, a.n - 16 * t);
        for (int e = u; e < live * (D / 4); e += 64 * kspl) {
            const int c = e / (D / 4), d = 4 * (e - c * (D / 4));
            float mm = ml[g0][16 * t + c][0], ll = 0.f;
            for (int x = 1; x < kspl; ++x) mm = fmaxf(mm, ml[g0 + x][16 * t + c][0]);
            float4_t r = {0.f, 0.f, 0.f, 0.f};
            for (int x = 0; x < kspl; ++x) {
                const float f = half_fall(ml[g0 + x][16 * t + c][0], mm);
                ll += ml[g0 + x][16 * t + c][1] * f * f;
                r += *reinterpret_cast<const float4_t*>(red[g0 + x] + c * ROW + d);
            }
            sink.put(a.c + 16 * t + c, d, r, over_sum<0>(ll));
            if (d == 0) sink.put_ml(a.c + 16 * t + c, mm, ll);
        }
    }
    if (w.chunks == 1 || p.join_apart) return;
    sink.join(min(2 * COLS, w.cols), reinterpret_cast<float4_t*>(&red[0][0]), reinterpret_cast<float(*)[2]>(&red[0][0] + 1024), &last);
}

template <typename E, int D, int NT>
__global__ __launch_bounds__(256) void kv8_join_kernel(KvAttnParams p) {
    __shared__ FewJoin lds;
    few_join<E, D, NT, 0>(p, lds);
}

template <typename E, int D, int NT>
static void run(const KvAttnShape& s, const KvAttnParams& p, hipStream_t st) {
    kv8_few_kernel<E, D, NT><<<dim3(p.Hkv, s.tiles, s.places), 256, 0, st>>>(p);
    if (p.join_apart) kv8_join_kernel<E, D, NT><<<dim3(p.Hkv, p.B, s.tiles * p.join_parts), 256, 0, st>>>(p);
}
template <typename E, int D>
static void go(const KvAttnShape& s, const KvAttnParams& p, hipStream_t st) {
    if constexpr (D <= 128)
        if (s.nt == 2) return run<E, D, 2>(s, p, st);
    run<E, D, 1>(s, p, st);
}

hipError_t launch_kv8_few(bool bf16, int D, const KvAttnParams& p, const KvAttnShape& s, hipStream_t st) {
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
