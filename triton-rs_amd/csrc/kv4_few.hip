// Attention over the 4-bit cache for few columns (at most 64 of a key/value head: single tokens, drafts):
// bound by the cache's bytes. The mathematics is in kv4_attn_body.h.
//
// The waves of a workgroup share their columns' keys, every second or fourth step of 32 each, and
// join through LDS. A wave brings its steps into an LDS ring of its own (buffer loads to LDS, no
// registers, no barrier), two steps in flight for each of the waves that its registers leave room for
// (three leave LDS for fewer workgroups: 68.1 against 61.5 us for the 4 sequences below). The keys
// of a sequence are split into chunks only as far as it takes to fill the device.
//
// Measured: 4 sequences of 65536 keys, 32 heads on 8 of D = 128, 65 us a call, 4.4 TB/s (a large copy
// reaches 4.8): 61 in this kernel, which issues vector instructions in half of its cycles, 5 in the join.
// 48 sequences of up to 4096 keys 39 us, 3.2 TB/s, every step as fast but a start and an end of some
// 6 us. One of 500 keys 9.5 us: launch, lengths, pages, first keys and the join of the waves one
// after another. 8 drafts of 5 tokens over windows of 4096 keys, 16 heads on 2 of D = 256, 27 us,
// 22 of them here with four steps a wave, likewise a chain.
#include "kv4_attn_body.h"
#include "kv_few.h"
#include "lds_dma.h"

namespace w4a16 {

template <int D>
struct FewShape {
    static constexpr int BLOCK = kv4_block_bytes(D);
    static constexpr int SLOTS = 2;
    static constexpr int RING = SLOTS * 2 * BLOCK;   // bytes of a wave
    // 16-byte loads of a block: whole waves of it, then the parameters
    static constexpr int FULL = D / 64, LOADS = FULL + 1;
    static constexpr int ROW = D + 4;                // LDS row of a column's result, in the ring's place
    static_assert(16 * ROW * 4 <= RING && 4096 + 2048 <= 4 * RING, "results of a wave, and what joins chunks, fit the rings");
};

// A block into LDS at dst: keys and values of D = 128 and 256 in the order in which lanes take them (16 bytes
// a lane), else as stored; then the parameters.
template <int D>
__device__ __forceinline__ void bring(unsigned char* dst, const unsigned char* src, int lane) {
    const i32x4_t rs = buffer_rsrc(src, kv4_block_bytes(D));
    if constexpr (D == 128) {
        dma16(rs, dst, (lane & 15) * 64 + (lane >> 4) * 16);
        dma16(rs, dst + 1024, 1024 + lane * 16);
    } else if constexpr (D == 256) {
#pragma unroll
        for (int x = 0; x < 2; ++x) dma16(rs, dst + 1024 * x, (lane & 15) * 128 + (lane >> 4) * 32 + 16 * x);
#pragma unroll
        for (int x = 0; x < 2; ++x) dma16(rs, dst + 2048 + 1024 * x, 2048 + lane * 32 + 16 * x);
    } else {
#pragma unroll
        for (int x = 0; x < D / 64; ++x) dma16(rs, dst + 1024 * x, 1024 * x + lane * 16);
    }
    if (lane < 8) dma16(rs, dst + 16 * D, 16 * D + lane * 16);
}

// This lane's words of keys (VAL = false) or values of a block in LDS.
template <int D, bool VAL>
__device__ __forceinline__ void take(uint32_t (&dst)[D / 32], const unsigned char* src, int lane) {
    if constexpr (D % 128 == 0) {
#pragma unroll
        for (int x = 0; x < D / 128; ++x) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(src + (VAL ? 8 * D : 0) + 1024 * x + lane * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) dst[4 * x + e] = v[e];
        }
    } else {
        const int off = VAL ? 8 * D + lane * (D / 8) : (lane & 15) * (D / 2) + (lane >> 4) * (D / 8);
#pragma unroll
        for (int x = 0; x < D / 64; ++x) {
            const u32x2 v = *reinterpret_cast<const u32x2*>(src + off + 8 * x);
            dst[2 * x] = v[0];
            dst[2 * x + 1] = v[1];
        }
    }
}

template <typename E, int D, int NT>
__global__ __launch_bounds__(256, kv4_few_per_cu(D, NT)) void kv4_few_kernel(KvAttnParams p) {
    typedef FewShape<D> S;
    typedef Kv4Cols<E, D, NT> C;
    constexpr int COLS = 16 * NT;
    __shared__ __align__(16) unsigned char ring[4][S::RING];
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
    const int stride = STEP << kshift, beg = (a.jlo & ~(STEP - 1)) + STEP * (wave & (kspl - 1)), end = a.jhi;
    unsigned char* const mine = ring[wave];
    const KvPages pages(p, w, S::BLOCK);
    int bad = 0;   // bits 2 slot + s: block s of a slot lies in no page
    auto fetch = [&](int slot, int at, int pa, int pb) {
        bring<D>(mine + slot * 2 * S::BLOCK, pages.block(pa, at >> 4), lane);
        bring<D>(mine + slot * 2 * S::BLOCK + S::BLOCK, pages.block(pb, (at >> 4) + 1), lane);
        const int f = (pages.ok(pa) ? 0 : 1) | (pages.ok(pb) ? 0 : 2);
        bad = (bad & ~(3 << (2 * slot))) | f << (2 * slot);
    };
#pragma unroll
    for (int s = 0; s < S::SLOTS; ++s) {
        const int at = beg + s * stride;
        if (at < end) fetch(s, at, pages.page(at >> 4), pages.page((at >> 4) + 1));
    }
    a.start(p, a.sizes());

    int slot = 0;
    // the pages of the step that takes this one's slot
    int pa = 0, pb = 0;
    if (beg + S::SLOTS * stride < end) {
        pa = pages.page((beg + S::SLOTS * stride) >> 4);
        pb = pages.page(((beg + S::SLOTS * stride) >> 4) + 1);
    }
    for (int j = beg; j < end; j += stride) {
        // this step's loads are done when only the later steps' are left
        if (j + (S::SLOTS - 1) * stride < end) wait_vmcnt<(S::SLOTS - 1) * 2 * S::LOADS>();
        else wait_vmcnt<0>();
        asm volatile("" ::: "memory");
        const unsigned char* src = mine + slot * 2 * S::BLOCK;
        uint32_t k[2][C::KW], v[2][C::KW], kc[2];
        u32x4 kp[2], vp[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const unsigned char* b = src + s * S::BLOCK;
            take<D, false>(k[s], b, lane);
            take<D, true>(v[s], b, lane);
            kc[s] = *reinterpret_cast<const uint32_t*>(b + 16 * D + 4 * col);
            kp[s] = *reinterpret_cast<const u32x4*>(b + 16 * D + 16 * kb);
            vp[s] = *reinterpret_cast<const u32x4*>(b + 16 * D + 64 + 16 * kb);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read: the slot is free
        const int here = (bad >> (2 * slot)) & 3;
        const int jn = j + S::SLOTS * stride;
        if (jn < end) {
            fetch(slot, jn, pa, pb);
            if (jn + stride < end) {
                pa = pages.page((jn + stride) >> 4);
                pb = pages.page(((jn + stride) >> 4) + 1);
            }
        }
        slot = slot + 1 == S::SLOTS ? 0 : slot + 1;

        const bool whole = j >= a.all_lo && j + STEP <= a.all_hi && j + STEP <= end && !here;
        if (!whole) {
            // tokens that no column sees may hold anything: their parameters become zeros
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (((here >> s) & 1) || j + 16 * s + 4 * kb + i >= end || j + 16 * s + 4 * kb + i < a.jlo) kp[s][i] = vp[s][i] = 0u;
        }
        float4_t acc[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = float4_t{0.f, 0.f, 0.f, 0.f};
        half2_t kz1[2], kz16[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            kz1[s] = zero1024(zeros_of(kc[s]));
            kz16[s] = zero64(zeros_of(kc[s]));
        }
#pragma unroll
        for (int x = 0; x < C::KW; ++x)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const half8_t f = key_operand(k[s][x], kz1[s], kz16[s]);
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[t][s] = mfma16x16x32(f, a.qf[t][x], acc[t][s]);
            }
        float ks[2][4], vs[2][4];
        uint32_t vmax = 0;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ks[s][i] = param_scale<E>(kp[s][i]) * a.kscale;
                vs[s][i] = value_scale<E>(vp[s][i]);
                vmax = max(vmax, __float_as_uint(vs[s][i]));
            }
        const float above = log2_above(vmax, a.least);
        a.uncommon(acc, ks, vs, above, whole, j, end, here, kb);
        half8_t pw[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float x[2][4];
            a.logits(t, x, acc[t], ks, vs, above, whole, j, end, here, kb);
            pw[t] = a.weights(t, x, vs);
        }
        half2_t vz1[4], vz16[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const uint32_t z = zeros_of(vp[y >> 1][2 * (y & 1)], vp[y >> 1][2 * (y & 1) + 1]);
            vz1[y] = zero1024(z);
            vz16[y] = zero64(z);
        }
#pragma unroll
        for (int g = 0; g < D / 64; ++g) {
            const uint32_t x[4] = {v[0][g], v[0][D / 64 + g], v[1][g], v[1][D / 64 + g]};
            auto product = [&](auto ei) {
                constexpr int e = decltype(ei)::value;
                const half8_t f = as_h8(value_pair<e>(x[0], vz1[0], vz16[0]), value_pair<e>(x[1], vz1[1], vz16[1]),
                                        value_pair<e>(x[2], vz1[2], vz16[2]), value_pair<e>(x[3], vz1[3], vz16[3]));
#pragma unroll
                for (int t = 0; t < NT; ++t) a.o[t][4 * g + e] = mfma16x16x32(f, pw[t], a.o[t][4 * g + e]);
            };
            product(std::integral_constant<int, 0>{});
            product(std::integral_constant<int, 1>{});
            product(std::integral_constant<int, 2>{});
            product(std::integral_constant<int, 3>{});
        }
    }
    a.finish();

    // the waves of a group join their shares of the keys
    const KvSink<E, D, VALUE_DOWN<E>> sink(p, w);
#pragma unroll
    for (int t = 0; t < NT; ++t)
        if (kb == 0) {
            ml[wave][16 * t + col][0] = a.m[t];
            ml[wave][16 * t + col][1] = a.l[t];
        }
    __syncthreads();
    const int u = threadIdx.x & (64 * kspl - 1);
    float* const red = reinterpret_cast<float*>(mine);
    constexpr int RING_FLOATS = S::RING / 4;
    const float* const reds = reinterpret_cast<const float*>(ring[g0]);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float top = ml[g0][16 * t + col][0];
        for (int x = 1; x < kspl; ++x) top = fmaxf(top, ml[g0 + x][16 * t + col][0]);
        const float f = __builtin_amdgcn_exp2f(a.m[t] - top);
        if (t) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int x = 0; x < C::VT; x += 4)
                *reinterpret_cast<float4_t*>(red + col * S::ROW + (4 * kb + i) * C::VT + x) =
                    float4_t{a.o[t][x][i], a.o[t][x + 1][i], a.o[t][x + 2][i], a.o[t][x + 3][i]} * f;
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
                r += *reinterpret_cast<const float4_t*>(reds + x * RING_FLOATS + c * S::ROW + d);
            }
            sink.put(a.c + 16 * t + c, d, r, over_sum<VALUE_DOWN<E>>(ll));
            if (d == 0) sink.put_ml(a.c + 16 * t + c, mm, ll);
        }
    }
    if (w.chunks == 1 || p.join_apart) return;
    sink.join(min(2 * COLS, w.cols), reinterpret_cast<float4_t*>(&ring[0][0]), reinterpret_cast<float(*)[2]>(&ring[0][4096]), &last);
}

template <typename E, int D, int NT>
__global__ __launch_bounds__(256) void kv4_join_kernel(KvAttnParams p) {
    __shared__ FewJoin lds;
    few_join<E, D, NT, VALUE_DOWN<E>>(p, lds);
}

template <typename E, int D, int NT>
static void run(const KvAttnShape& s, const KvAttnParams& p, hipStream_t st) {
    kv4_few_kernel<E, D, NT><<<dim3(p.Hkv, s.tiles, s.places), 256, 0, st>>>(p);
    if (p.join_apart) kv4_join_kernel<E, D, NT><<<dim3(p.Hkv, p.B, s.tiles * p.join_parts), 256, 0, st>>>(p);
}
template <typename E, int D>
static void go(const KvAttnShape& s, const KvAttnParams& p, hipStream_t st) {
    if constexpr (D <= 128)
        if (s.nt == 2) return run<E, D, 2>(s, p, st);
    run<E, D, 1>(s, p, st);
}

hipError_t launch_kv4_few(bool bf16, int D, const KvAttnParams& p, const KvAttnShape& s, hipStream_t st) {
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
