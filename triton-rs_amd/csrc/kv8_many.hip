// Attention over the 8-bit cache for many columns (prompts, chunks of them): bound by the matrix and
// vector instructions, of which one wave's overlap little with another's. The mathematics is in kv8_attn_body.h.
//
// A workgroup of four waves takes 128 columns, 32 a wave, and walks the keys 64 at a time: each wave turns
// a block of 16 tokens into operands once for all four, in LDS and in the order in which lanes take them (16
// bytes a lane, no bank conflicts), while the step before is computed from the other half of the LDS: one
// barrier a step. The bytes come a step ahead into registers.
//
// Measured: 1024 queries over 32768 keys, 32 heads on 8 of D = 128, 600 to 625 us (0.88 PFLOP/s, matrix cores busy 42 %, vector unit
// 51); a prompt of 2048 60 us, of 512 20. 64 columns a wave, one wave a SIMD, halve what is read from LDS and took 966
// us, with the products and the vector instructions beside them in an order of their own 1580 (registers beyond 256 are moved).
#include "kv8_attn_body.h"
#include "kv_many.h"

namespace w4a16 {

// The 32 x 32 x 16 product: lane l has row (or column) l % 32 of an operand at k = 8 (l / 32) + (0..7), and column l % 32 of the
// result at rows 8 (i / 4) + 4 (l / 32) + i % 4. The vector unit runs beside it (64 multiplications and additions of one
// wave and the products of another: 164 ns, 131 and 125 alone; beside as much work in 16 x 16 x 32 products 200).
__device__ __forceinline__ float16_t mfma32x32x16(half8_t a, half8_t b, float16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float16_t mfma32x32x16(bf16x8_t a, bf16x8_t b, float16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

template <typename E, int D>
struct ManyLds {
    static constexpr int KW = D / 16, VT = D / 32;
    typename vec8<E>::type k[2][KW][64];   // pair of blocks, 16 dimensions, lane (token l % 32 of the pair)
    half8_t v[4][VT][64];                  // block, 32 dimensions, lane (its quads l / 32 and 2 + l / 32 of tokens)
    Kv8Scale scale[4];
    int live[4];                           // tokens of a block that there are (0 or less: none)
};

// A block (of this wave) as this lane takes it.
template <int D>
struct Packed {
    u32x4 k[D / 64], v[D / 64];
    u32x3 tail;
};

// Piece i of UNPACK_PIECES of block b of a step into LDS; its tokens [dead, live) (the others' bytes may be anything)
template <int D>
constexpr int UNPACK_PIECES = 6 * (D / 64);
template <typename E, int D>
__device__ __forceinline__ void unpack_piece(ManyLds<E, D>& s, const Packed<D>& t, int i, uint32_t mask, int b, int lane) {
    const int r = lane & 15, quad = lane >> 4, g = i / 6, h = i % 6;
    if (h < 2) {
        s.k[b >> 1][4 * g + quad][16 * (b & 1) + r + 32 * h] = operand8<E>(t.k[g][2 * h], t.k[g][2 * h + 1]);
    } else {   // dimension r D / 16 + x, x = 4 g + e, is row r + 16 (x % 2) of tile x / 2
        const int e = h - 2;
        const uint32_t w = t.v[g][e] & mask;
        reinterpret_cast<u32x2*>(&s.v[b][2 * g + e / 2][r + 32 * (quad & 1) + 16 * (e & 1)])[quad >> 1] =
            u32x2{from_e4m3<half_t, false>(w), from_e4m3<half_t, true>(w)};
    }
}
__device__ __forceinline__ uint32_t live_bytes(int dead, int live, int lane) { return dead <= 0 && live >= 16 ? ~0u : token_bytes(dead, live, lane >> 4); }
template <typename E, int D>
__device__ __forceinline__ void unpack_scale(ManyLds<E, D>& s, const Packed<D>& t, int dead, int live, float factor, int b, int lane) {
    if (lane == 0) {
        s.scale[b] = Kv8Scale::of(t.tail, factor, live > 0 && dead < 16);
        s.live[b] = live;
    }
}
template <typename E, int D>
__device__ __forceinline__ void unpack(ManyLds<E, D>& s, const Packed<D>& t, int dead, int live, float factor, int b, int lane) {
    const uint32_t mask = live_bytes(dead, live, lane);
#pragma unroll
    for (int i = 0; i < UNPACK_PIECES<D>; ++i) unpack_piece<E, D>(s, t, i, mask, b, lane);
    unpack_scale<E, D>(s, t, dead, live, factor, b, lane);
}

__device__ __forceinline__ float half_max(float v) {   // over a column's two lanes, 32 apart
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The largest of three, one of which is not NaN. (The compiler's own first quiets what it has from another block, an instruction
// an operand.)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// A wave's 32 columns, column lane % 32 in a lane; as Kv8Cols, whose comments hold here.
template <typename E, int D>
struct ManyCols {
    typedef typename vec8<E>::type vec_t;
    static constexpr int KW = D / 16, VT = D / 32;
    float16_t o[VT];       // dimension r D / 16 + 2 y + z, r + 16 z = 8 (i / 4) + 4 (lane / 32) + i % 4, in o[y][i]
    vec_t qf[KW];          // dimensions 16 x + 8 (lane / 32) + (0..7)
    float m, l, most;
    int c, n, lo, hi, jlo, jhi, all_lo, all_hi;

    __device__ __forceinline__ void load(const KvAttnParams& p, const KvItem& w, int first_col, int lane) {
        c = first_col;
        n = min(32, w.n * p.G - c);
        const int col = lane & 31, r = c + col, i = w.n == 1 ? 0 : r / p.G;
        const bool in = col < n;
        hi = in ? w.see_hi(p, i) : 0;
        lo = in ? w.see_lo(p, i) : 0;
        const uint16_t* src = static_cast<const uint16_t*>(p.q) + (size_t)(w.q0 + i) * p.q_st + (size_t)(w.h * p.G + r - i * p.G) * p.q_sh + 8 * (lane >> 5);
        constexpr uint32_t inf = __is_same(E, half_t) ? 0x7C00u : 0x7F80u;
#pragma unroll
        for (int x = 0; x < KW; ++x) {
            u32x4 v = {0, 0, 0, 0};
            if (in) v = *reinterpret_cast<const u32x4*>(src + 16 * x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {   // infinities become NaN
                const uint32_t u = v[e], a = u & 0x7FFFu, b = (u >> 16) & 0x7FFFu;
                v[e] = u | (a < inf ? 0u : 0x7FFFu) | (b < inf ? 0u : 0x7FFF0000u);
            }
            qf[x] = __builtin_bit_cast(vec_t, v);
        }
        const int i0 = w.n == 1 ? 0 : c / p.G, i1 = w.n == 1 ? 0 : (c + max(n, 1) - 1) / p.G;
        jlo = max(w.k0, w.see_lo(p, i0));
        jhi = n > 0 ? min(w.k1, w.see_hi(p, i1)) : 0;
        all_lo = w.see_lo(p, i1);
        all_hi = w.see_hi(p, i0);
        m = l = 0.f;
        most = -INFINITY;
#pragma unroll
        for (int y = 0; y < VT; ++y)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[y][e] = 0.f;
    }

    // Tokens j + 8 (i / 4) + 4 (lane / 32) + i % 4 of 32 from j on: [from, to) of the lane's 16 logits
    __device__ __forceinline__ void logits(float (&x)[16], const float16_t& acc, const Kv8Scale (&s)[2], int from, int to) const {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i >= from && i < to) x[i] = __builtin_fmaf(acc[i], s[i / 8].key, s[i / 8].value - m);
    }
    // What is not seen, or not finite. whole: nothing of that.
    __device__ __forceinline__ void mask(float (&x)[16], const Kv8Scale (&s)[2], bool whole, int j, int end, int bad, int lane) {
        if (!whole) {
            int at = j + 4 * (lane >> 5);
            asm volatile("" : "+v"(at), "+s"(bad));   // (else kept over the loop: every token's distances, in registers)
            const int from = lo - at, to = min(hi, end) - at;
            uint32_t hit = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int t = 8 * (i / 4) + i % 4, b = i / 8, bit = (t + 4 * (lane >> 5)) & 15;
                const bool in = (t >= from) & (t < to) & !((bad >> b) & 1);
                if ((s[b].nan >> bit) & 1) x[i] = __builtin_nanf("");
                if (!in) x[i] = -INFINITY;
                hit |= in ? (s[b].nan >> (16 + bit)) & 1 : 0u;
            }
            if ((s[0].nan | s[1].nan) >> 16) {   // a value row of NaN makes those columns NaN that see it
                const float add = half_max(hit ? 1.f : 0.f) > 0.f ? __builtin_nanf("") : 0.f;
#pragma unroll
                for (int y = 0; y < VT; ++y)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[y][i] += add;
            }
        }
    }
    // The reference follows; how the lane's sums take a block's weights in back.
    __device__ __forceinline__ void follow(float (&x)[16], float (&back)[2], const Kv8Scale (&s)[2]) {
        float high[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            high[b] = max3(max3(x[8 * b], x[8 * b + 1], x[8 * b + 2]), max3(x[8 * b + 3], x[8 * b + 4], x[8 * b + 5]), max3(x[8 * b + 6], x[8 * b + 7], x[8 * b + 7]));
            back[b] = s[b].back;
        }
        float top = fmaxf(high[0], high[1]);
        if (__any((top > most) | (fminf(high[0], high[1]) < KV8_LOW))) {   // rare after the first steps
            top = half_max(top);
            const bool up = top > most;
            const float by = up ? top - (KV8_MOST - KV8_ROOM) : 0.f;
            const float fall = most == -INFINITY ? 0.f : half_fall(0.f, by);
            m += by;
            l = l * fall * fall;
#pragma unroll
            for (int y = 0; y < VT; ++y)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[y][i] *= fall * fall;
            most = up ? KV8_MOST : most;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const bool alone = high[b] - by < KV8_LOW;
                float p = 0.f;
#pragma unroll
                for (int i = 8 * b; i < 8 * b + 8; ++i) {
                    x[i] -= by;
                    p += __builtin_amdgcn_exp2f(x[i] - s[b].value);
                }
                l += alone ? p : 0.f;
                back[b] = alone ? 0.f : back[b];
            }
        }
    }
    // Weights [from, to) of the lane's 16; a block's as operand; the sum of p_j.
    __device__ __forceinline__ static void weights(float (&x)[16], int from, int to) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i >= from && i < to) x[i] = __builtin_amdgcn_exp2f(x[i]);
    }
    __device__ __forceinline__ static half8_t operand(const float (&w)[16], int b) {
        half8_t h;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = (half_t)w[8 * b + i];
        return h;
    }
    __device__ __forceinline__ void sum(const float (&w)[16], const float (&back)[2], int b) {
        const float* f = w + 8 * b;
        l = __builtin_fmaf(((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7])), back[b], l);
    }
    __device__ __forceinline__ void finish() {
        l = half_sum(l);
        if (most == -INFINITY && l == 0.f) m = -FLT_MAX;
    }
    // Rows of the result: quad xq (four dimensions in a row) of rr-th row r
    __device__ __forceinline__ static int row(int rr, int lane) { return 8 * (rr / 4) + 4 * (lane >> 5) + rr % 4; }
    __device__ __forceinline__ float4_t quad(int rr, int xq) const {
        return float4_t{o[2 * xq][rr], o[2 * xq][rr + 8], o[2 * xq + 1][rr], o[2 * xq + 1][rr + 8]};
    }
    // Partial results as lanes have them: number of a quad, and place of quad e
    static constexpr int XQ = D / 64;
    __device__ __forceinline__ static int lane_quad(int wave, int rr, int xq, int lane) { return ((wave * 8 + rr) * XQ + xq) * 64 + lane; }
    __device__ __forceinline__ static void lane_place(int e, int& c, int& d) {
        const int lane = e & 63, q = e >> 6, xq = q % XQ, u = q / XQ;
        c = 32 * (u >> 3) + (lane & 31);
        d = row(u & 7, lane) * (D / 16) + 4 * xq;
    }
};

// What stands before it is issued before what stands behind.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }
template <typename E, int D, int GROUPS>
__global__ __launch_bounds__(256 * GROUPS, kv8_many_simd_waves(D, GROUPS)) void kv8_many_kernel(KvAttnParams p) {
    constexpr int COLS = 32, STEP = MANY_STEP, ALL = STEP * GROUPS;
    typedef ManyCols<E, D> C;
    __shared__ ManyLds<E, D> lds[2][GROUPS];
    KvItem w;
    if (!many_item(p, blockIdx.z, w)) return;
    // wave `wave` of group `group`: the group takes every GROUPS-th step of the keys
    const int lane = threadIdx.x & 63, number = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = number & 3, group = number >> 2;
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
        // (only a first step holds tokens before what its columns see)
        unpack<E, D>(lds[0][group], t, w.see_lo(p, w.n <= 1 ? 0 : w.c0 / p.G) - (w.k0 + STEP * group + 16 * wave), live, p.scale_log2, wave, lane);
        fetch(w.k0 + ALL);
    }
    __syncthreads();
    int buf = 0;
    // Two waves a SIMD (D <= 128): the next step is unpacked beside this one's products of keys, a half step's share each, and the
    // instructions of the second product stand in this order (1024 queries over 32768 keys of 8 heads 618 us, 637 in the compiler's).
    // One wave: all of it first, so that the bytes of the step behind it are a step ahead (2048 of D = 256 119 us, 124).
    constexpr bool BESIDE = D <= 128;
    constexpr int PIECES = UNPACK_PIECES<D> / 2;   // of a half step
    for (int j = w.k0; j < w.k1; j += ALL, buf ^= 1) {
        const ManyLds<E, D>& s = lds[buf][group];
        ManyLds<E, D>& into = lds[buf ^ 1][group];   // the next step's (behind the last: that of no step)
        const uint32_t bytes = live_bytes(0, live, lane);
        if constexpr (!BESIDE)
            if (j + ALL < w.k1) {
                unpack<E, D>(into, t, 0, live, p.scale_log2, wave, lane);
                fetch(j + 2 * ALL);
            }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int jh = j + STEP * group + 32 * half;
            auto piece = [&](int i) { unpack_piece<E, D>(into, t, half * PIECES + i, bytes, wave, lane); };
            auto rest = [&] {
                if (half == 0) return;   // (the first half's share stands there)
                unpack_scale<E, D>(into, t, 0, live, p.scale_log2, wave, lane);
                fetch(j + 2 * ALL);
            };
            if (jh >= a.jhi || jh + 32 <= a.jlo) {   // none of this wave's columns sees these
                if constexpr (BESIDE) {
#pragma unroll
                    for (int i = 0; i < PIECES; ++i) piece(i);
                    rest();
                }
                continue;
            }
            float16_t acc;
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[i] = 0.f;
            // operands from LDS all at once, ahead of what takes them: one wait instead of eight
            typename C::vec_t kf[C::KW];
            half8_t vf[2][C::VT];
            Kv8Scale sc[2] = {s.scale[2 * half], s.scale[2 * half + 1]};
            const int live0 = s.live[2 * half], live1 = s.live[2 * half + 1];
#pragma unroll
            for (int x = 0; x < C::KW; ++x) kf[x] = s.k[half][x][lane];
            in_order();
            const int bad = __builtin_amdgcn_readfirstlane((live0 <= 0 ? 1 : 0) | (live1 <= 0 ? 2 : 0));
            sc[0].nan = __builtin_amdgcn_readfirstlane(sc[0].nan);
            sc[1].nan = __builtin_amdgcn_readfirstlane(sc[1].nan);
            // (& and no &&, which would be a branch ahead of the products: D = 192, 1024 over 16384 378 us, 340 so)
            const bool whole = (jh >= a.all_lo) & (jh + 32 <= a.all_hi) & (jh + 32 <= a.jhi) & !bad & !(sc[0].nan | sc[1].nan);
#pragma unroll
            for (int x = 0; x < C::KW; ++x) {
                acc = mfma32x32x16(kf[x], a.qf[x], acc);
                if constexpr (BESIDE) {
                    in_order();
#pragma unroll
                    for (int i = x * PIECES / C::KW; i < (x + 1) * PIECES / C::KW; ++i) piece(i);
                    in_order();
                }
            }
            if constexpr (BESIDE) rest();
            float x[16], back[2];
            a.logits(x, acc, sc, 0, 16);
            a.mask(x, sc, whole, jh, a.jhi, bad, lane);
            a.follow(x, back, sc);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int y = 0; y < C::VT; ++y) vf[b][y] = s.v[2 * half + b][y][lane];
            in_order();
            if constexpr (BESIDE) {
                C::weights(x, 0, 8);
                half8_t pw = C::operand(x, 0);
#pragma unroll
                for (int y = 0; y < C::VT; ++y) {
                    a.o[y] = mfma32x32x16(vf[0][y], pw, a.o[y]);
                    in_order();
                    C::weights(x, 8 + y * 8 / C::VT, 8 + (y + 1) * 8 / C::VT);
                    in_order();
                }
                pw = C::operand(x, 1);
#pragma unroll
                for (int y = 0; y < C::VT; ++y) {
                    a.o[y] = mfma32x32x16(vf[1][y], pw, a.o[y]);
                    in_order();
                    if (y < 2) a.sum(x, back, y);
                    in_order();
                }
            } else {
                C::weights(x, 0, 16);
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const half8_t pw = C::operand(x, b);
                    a.sum(x, back, b);
#pragma unroll
                    for (int y = 0; y < C::VT; ++y) a.o[y] = mfma32x32x16(vf[b][y], pw, a.o[y]);
                }
            }
        }
        __syncthreads();
    }
    a.finish();

    if constexpr (GROUPS == 2) {   // the second group's share of the keys to the first
        float4_t* const o = reinterpret_cast<float4_t*>(&lds[0][0]) + wave * (4 * C::VT) * 64;
        float* const mls = reinterpret_cast<float*>(reinterpret_cast<float4_t*>(&lds[0][0]) + 4 * (4 * C::VT) * 64) + wave * 128;
        static_assert(4 * 4 * C::VT * 64 * 16 + 4 * 128 * 4 <= sizeof(lds), "results of four waves fit");
        if (group) {
            mls[lane] = a.m;
            mls[64 + lane] = a.l;
#pragma unroll
            for (int y = 0; y < C::VT; ++y)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[(4 * y + e) * 64 + lane] = float4_t{a.o[y][4 * e], a.o[y][4 * e + 1], a.o[y][4 * e + 2], a.o[y][4 * e + 3]};
        }
        __syncthreads();
        if (group) return;
        const float m1 = mls[lane], mm = fmaxf(a.m, m1);
        const float h0 = half_fall(a.m, mm), h1 = half_fall(m1, mm), f0 = h0 * h0, f1 = h1 * h1;
        a.m = mm;
        a.l = a.l * h0 * h0 + mls[64 + lane] * h1 * h1;
#pragma unroll
        for (int y = 0; y < C::VT; ++y)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float4_t u = o[(4 * y + e) * 64 + lane];
#pragma unroll
                for (int i = 0; i < 4; ++i) a.o[y][4 * e + i] = a.o[y][4 * e + i] * f0 + u[i] * f1;
            }
    }
    const KvSink<E, D, 0> sink(p, w);
    const int col = lane & 31;
    const float inv = over_sum<0>(a.l);
#pragma unroll
    for (int rr = 0; rr < 8; ++rr)
#pragma unroll
        for (int xq = 0; xq < C::XQ; ++xq) {
            const float4_t v = a.quad(rr, xq);
            // (chunks of partial results as they lie: 1 KiB a store and wave)
            if (w.chunks > 1) {
                st_partial4<SCOPE_DEVICE>(sink.part + 4 * C::lane_quad(wave, rr, xq, lane), v);
            } else if (col < a.n) {
                if constexpr (C::XQ % 2 == 0) {   // 16 bytes a store
                    if (xq % 2) sink.out8(a.c + col, C::row(rr, lane) * (D / 16) + 4 * (xq - 1), a.quad(rr, xq - 1), v, inv);
                } else {
                    sink.out(a.c + col, C::row(rr, lane) * (D / 16) + 4 * xq, v, inv);
                }
            }
        }
    if (lane < 32 && col < a.n) sink.put_ml(a.c + col, a.m, a.l);
}

template <typename E, int D>
__global__ __launch_bounds__(256) void kv8_many_join_kernel(KvAttnParams p) {
    __shared__ float ml[128][2];
    many_join<E, D, 0>(p, &ml[0][0], [](int e, int& c, int& d) { ManyCols<E, D>::lane_place(e, c, d); });
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
