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
#include "lds_dma.h"

namespace w4a16 {

constexpr int STEP = 32;   // keys of a step

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

__device__ __forceinline__ unsigned wave_sum(int v) { return (unsigned)__builtin_amdgcn_readlane(wave_sums(v), 63); }
__device__ __forceinline__ int wave_max(int v) { return __builtin_amdgcn_readlane(wave_scan(v, [](int a, int b) { return max(a, b); }), 63); }

// Chunks of `steps` steps of keys in chunks of c 128 (4 c steps); -1: no columns here. Up to 512 keys stay whole, as a
// chunk more costs its partial results' way to the last one and back: one sequence, 8 heads of D = 128, 500 keys 9.0 us
// whole, 9.8 in chunks, 700 keys 11.0, 9.4; 4 drafts of 5 tokens, 8 heads a group, 500 keys 19.8, 20.5, 700 23.5, 17.2.
__device__ __forceinline__ int few_chunks(int steps, int c) {
    return steps < 0 ? 0 : steps <= max(KV4_WHOLE_KEYS / STEP, 4 * c) ? 1 : (steps + 4 * c - 1) / (4 * c);
}

// The length of chunks, in 128 keys, for sequences of `sum` steps together and `most` at most, total(c) their number:
// at most p.budget of them, whatever the lengths. Keys / budget or keys / (budget - B / 2) where that is enough, else
// keys / (budget - B) (the budget is twice B or more); or all sequences whole where that is estimated to take no longer.
template <typename F>
__device__ __forceinline__ int few_length(const Kv4AttnParams& p, unsigned sum, int most, F total) {
    int c = 1;
    unsigned n = p.budget;
    for (int rest = 0; rest <= 4; rest += 2) {   // no remainders, half a chunk a sequence, one a sequence
        const unsigned room = 4 * p.budget - rest * p.B;
        c = (int)max(1u, (sum + room - 1) / room);
        if (rest == 4) break;
        const unsigned t = total(c);
        if (t <= (unsigned)p.budget) {
            n = t;
            break;
        }
    }
    // In steps of a full device (0.85 us at D = 128, the only one these were measured at): a round of workgroups costs 6 besides its steps, a step of one
    // workgroup alone 0.45, joining 7. Whole and in two, 8 heads of D = 128: 128 sequences of 1000 keys 34, 49 us, 256
    // of 900 58, 103; 48 of 4096 56, 54.
    auto cost = [&](unsigned chunks, int steps) {
        const float rounds = (float)((chunks + p.at_once - 1) / p.at_once);
        return 6.f * rounds + fmaxf(0.45f * rounds * (float)steps, (float)sum / (float)p.at_once);
    };
    if (__builtin_amdgcn_readfirstlane(cost(p.B, most) <= cost(n, min(4 * c, most)) + 7.f)) c = max(c, (most + 3) / 4);
    return c;
}

// What the waves of a workgroup tell each other of more than 64 sequences.
struct FewFind {
    unsigned total[4][4];   // per pass and wave
    int most[4];
    int hit[3];             // sequence (-1: none), its first chunk's number, its chunks
};

// The chunks of all sequences for one head and tile of columns stand in a row; workgroup u of 256 threads takes the
// u-th. With by_seq, sequence u's first chunk instead. A lane a sequence, up to 64; a thread several, beyond (their
// order in the row is that of the threads).
template <int WG_COLS>
__device__ __forceinline__ bool few_item(const Kv4AttnParams& p, int tile, int u, bool by_seq, Kv4Item& w, FewFind& find) {
    w.h = blockIdx.x;
    int lo = 0, hi = 0;
    if (p.whole) {   // sequence u, in one chunk
        w.sequence<WG_COLS, STEP>(p, u, tile * WG_COLS, lo, hi);
        w.take(0, 1, 0, lo, hi);
        w.at = w.slot = 0;   // (no partial results)
        return w.cols > 0;
    }
    Kv4Item mine;
    auto look = [&](int b) {   // steps of sequence b, -1 without columns
        mine.sequence<WG_COLS, STEP>(p, min(b, p.B - 1), tile * WG_COLS, lo, hi);
        return b < p.B && mine.cols > 0 ? (hi - lo + STEP - 1) / STEP : -1;
    };
    int at, chunks, c;
    if (p.B <= 64) {
        const int lane = threadIdx.x & 63, steps = look(lane);
        c = few_length(p, wave_sum(max(steps, 0)), wave_max(max(steps, 0)), [&](int c) { return wave_sum(few_chunks(steps, c)); });
        const int here = few_chunks(steps, c), upto = wave_sums(here);
        const uint64_t who = __ballot(by_seq ? lane == u && here > 0 : upto - here <= u && u < upto);
        if (!who) return false;
        const int l = __builtin_ctzll(who);
        auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
        at = of(upto - here);
        chunks = of(here);
        w.b = l;
        w.q0 = of(mine.q0);
        w.n = of(mine.n);
        w.len = of(mine.len);
        w.first = of(mine.first);
        w.c0 = tile * WG_COLS;
        w.cols = of(mine.cols);
        lo = of(lo);
        hi = of(hi);
    } else {
        const int wave = threadIdx.x >> 6;
        constexpr int HELD = 4;   // of a thread's sequences, in registers, their loads in flight together
        int held[HELD];
#pragma unroll
        for (int g = 0; g < HELD; ++g) held[g] = look(256 * g + threadIdx.x);
        auto each = [&](auto f) {
#pragma unroll
            for (int g = 0; g < HELD; ++g) f(256 * g + (int)threadIdx.x, held[g]);
            for (int b = 256 * HELD + threadIdx.x; b < p.B; b += 256) f(b, look(b));
        };
        auto all = [&](int pass, unsigned v) {   // sum over the workgroup
            v = wave_sum((int)v);
            if ((threadIdx.x & 63) == 0) find.total[pass][wave] = v;
            __syncthreads();
            return find.total[pass][0] + find.total[pass][1] + find.total[pass][2] + find.total[pass][3];
        };
        unsigned mine_sum = 0;
        int mine_most = 0;
        each([&](int, int steps) {
            mine_sum += max(steps, 0);
            mine_most = max(mine_most, steps);
        });
        auto mine_chunks = [&](int c) {
            unsigned n = 0;
            each([&](int, int steps) { n += few_chunks(steps, c); });
            return n;
        };
        mine_most = wave_max(mine_most);
        if ((threadIdx.x & 63) == 0) find.most[wave] = mine_most;
        if (threadIdx.x == 0) find.hit[0] = -1;
        const unsigned sum = all(0, mine_sum);
        const int most = max(max(find.most[0], find.most[1]), max(find.most[2], find.most[3]));
        int pass = 0;
        c = __builtin_amdgcn_readfirstlane(few_length(p, sum, most, [&](int c) { return all(++pass, mine_chunks(c)); }));
        const unsigned n = mine_chunks(c), upto = (unsigned)wave_sums((int)n);
        all(3, n);
        unsigned first = upto - n;   // number of this thread's first chunk
        for (int x = 0; x < wave; ++x) first += find.total[3][x];
        if (by_seq ? (u & 255) == (int)threadIdx.x : first <= (unsigned)u && (unsigned)u < first + n)
            each([&](int b, int steps) {
                const unsigned here = few_chunks(steps, c);
                if (by_seq ? b == u && here > 0 : first <= (unsigned)u && (unsigned)u < first + here) {
                    find.hit[0] = b;
                    find.hit[1] = (int)first;
                    find.hit[2] = (int)here;
                }
                first += here;
            });
        __syncthreads();
        const int b = __builtin_amdgcn_readfirstlane(find.hit[0]);
        if (b < 0) return false;
        at = __builtin_amdgcn_readfirstlane(find.hit[1]);
        chunks = __builtin_amdgcn_readfirstlane(find.hit[2]);
        w.sequence<WG_COLS, STEP>(p, b, tile * WG_COLS, lo, hi);
    }
    w.at = ((size_t)tile * p.B + w.b) * p.Hkv + w.h;
    w.slot = ((size_t)tile * p.Hkv + w.h) * p.places + at;
    w.take(by_seq ? 0 : u - at, chunks, 128 * c, lo, hi);
    return true;
}

template <typename E, int D, int NT>
__global__ __launch_bounds__(256, kv4_few_per_cu(D, NT)) void kv4_few_kernel(Kv4AttnParams p) {
    typedef FewShape<D> S;
    typedef Kv4Cols<E, D, NT> C;
    constexpr int COLS = 16 * NT;
    __shared__ __align__(16) unsigned char ring[4][S::RING];
    __shared__ float ml[4][COLS][2];
    __shared__ int last;
    __shared__ FewFind find;
    Kv4Item w;
    if (!few_item<2 * COLS>(p, blockIdx.y, blockIdx.z, false, w, find)) return;
    // one group of columns, its keys over four waves, or two over two
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kshift = w.cols <= COLS ? 2 : 1, kspl = 1 << kshift, g0 = wave & ~(kspl - 1);
    const int col = lane & 15, kb = lane >> 4;

    C a;
    a.load(p, w, w.c0 + (wave >> kshift) * COLS, lane);
    const int stride = STEP << kshift, beg = (a.jlo & ~(STEP - 1)) + STEP * (wave & (kspl - 1)), end = a.jhi;
    unsigned char* const mine = ring[wave];
    const Kv4Pages pages(p, w, S::BLOCK);
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
    const Kv4Sink<E, D> sink(p, w);
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
            sink.put(a.c + 16 * t + c, d, r, over_sum<E>(ll));
            if (d == 0) sink.put_ml(a.c + 16 * t + c, mm, ll);
        }
    }
    if (w.chunks == 1 || p.join_apart) return;
    sink.join(min(2 * COLS, w.cols), reinterpret_cast<float4_t*>(&ring[0][0]), reinterpret_cast<float(*)[2]>(&ring[0][4096]), &last);
}

// Joins the chunks of one sequence and head where that is more than one workgroup does in passing: 64 quads of
// values a workgroup, a quarter of the chunks a wave.
template <typename E, int D, int NT>
__global__ __launch_bounds__(256) void kv4_join_kernel(Kv4AttnParams p) {
    __shared__ float4_t vals[256];
    __shared__ float ml[256][2];
    __shared__ FewFind find;
    constexpr int COLS = 32 * NT;
    Kv4Item w;
    const int tile = p.tiles == 1 ? 0 : blockIdx.z / p.join_parts;
    if (!few_item<COLS>(p, tile, blockIdx.y, true, w, find) || w.chunks == 1) return;
    const Kv4Sink<E, D> sink(p, w);
    const int e = (blockIdx.z - tile * p.join_parts) * 64 + (threadIdx.x & 63);
    sink.join_quads(e, threadIdx.x >> 6, 4, 64, e < w.cols * (D / 4), vals, ml);
}

template <typename E, int D, int NT>
static void run(const Kv4AttnShape& s, const Kv4AttnParams& p, hipStream_t st) {
    kv4_few_kernel<E, D, NT><<<dim3(p.Hkv, s.tiles, s.places), 256, 0, st>>>(p);
    if (p.join_apart) kv4_join_kernel<E, D, NT><<<dim3(p.Hkv, p.B, s.tiles * p.join_parts), 256, 0, st>>>(p);
}
template <typename E, int D>
static void go(const Kv4AttnShape& s, const Kv4AttnParams& p, hipStream_t st) {
    if constexpr (D <= 128)
        if (s.nt == 2) return run<E, D, 2>(s, p, st);
    run<E, D, 1>(s, p, st);
}

hipError_t launch_kv4_few(bool bf16, int D, const Kv4AttnParams& p, const Kv4AttnShape& s, hipStream_t st) {
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
