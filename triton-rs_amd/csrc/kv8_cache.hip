// Rows of keys and values into the 8-bit cache (kv8.h), rotated on the way where asked, and back.
//
// A block's scale is the smallest power of two (2^-60 at least) of which 448 are its largest magnitude or more, so
// x / s is exact and a byte is x / s rounded to e4m3 once. Rows are appended: a block that already holds tokens of
// the sequence keeps its scale, or raises it to what the new rows need and takes the older bytes down by that power
// of two, which is exact but for what e4m3 holds as subnormals (below 2^-6 s).
//
// Bound by memory: 4 D bytes of a token's rows in, 2 D out. A workgroup takes a block (16 tokens) of some heads, so no two
// write one scale. Rows pass through LDS; then a thread has 16 bytes of the block, of keys 16 dimensions of
// a token, of values four tokens of four dimensions. Queries are rotated by workgroups of their own in the same launch (as
// one of rope.hip's they took 4 to 10 us more, start and end).
//
// Measured (rows from memory), 8 heads of D = 128: 8192 tokens 15.2 us (50 MB, 3.3 TB/s), keys rotated on the way 21.8, and 32
// heads of queries 46 (184 MB, 4.0 TB/s); 48 tokens of 48 sequences 4.4
// and 5.3; 8192 tokens read 11.6 (4.3 TB/s). What is left is registers: 77 and 91 of a thread leave six and five waves a SIMD (in 64
// it spills: 28 us), the next head's rows on their way beside this one's cost a wave and 1 us.
#include "kv8.h"
#include "kv_attn_body.h"
#include "rotate.h"

namespace w4a16 {

__device__ __forceinline__ float byte_f32(uint32_t w, int i) {   // byte i of w, e4m3
    return __builtin_amdgcn_cvt_f32_fp8((int)(w >> (8 * i)), 0);
}
// Four bytes under a scale of `ratio` times what they stand for.
__device__ __forceinline__ uint32_t rescale(uint32_t w, float ratio) {
    return to_e4m3(byte_f32(w, 0) * ratio, byte_f32(w, 1) * ratio, byte_f32(w, 2) * ratio, byte_f32(w, 3) * ratio);
}

// The largest of 16 lanes' numbers (lanes 16 i ..), all of which are active.
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, false));   // rotated by 8, 4, 2, 1 lanes
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xF, 0xF, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xF, 0xF, false));
}

// The new tokens of sequence b: rows q0.. of the call at positions [lo, hi) of the sequence; row of position lo.
struct Append { int lo, hi, row; };
__device__ __forceinline__ Append append(const Kv8WriteParams& p, int b) {
    const int* cu = p.cu_q ? p.cu_q + b : p.kv_lens;
    const int kv = p.kv_lens[b], q0 = p.cu_q ? min(max(cu[0], 0), p.T) : b, q1 = p.cu_q ? min(max(cu[1], 0), p.T) : b + 1;
    const int n = min(q1 - q0, p.max_q);
    if (n <= 0 || kv <= 0 || kv > (1 << 30)) return {0, 0, 0};
    const int first = kv - (q1 - q0);
    const long long cap = (long long)p.pages_per_seq << p.page_shift;
    const int lo = max(first, 0), hi = (int)min((long long)first + n, cap);
    return {lo, hi, q0 + lo - first};
}
__device__ __forceinline__ int append_blocks(Append a) { return a.hi > a.lo ? ((a.hi - 1) >> 4) - (a.lo >> 4) + 1 : 0; }

// Block `item` of all sequences' new tokens (each sequence's stand together): sequence and its number there.
__device__ __forceinline__ bool find_block(const Kv8WriteParams& p, int per_seq, int item, int& b, int& i, Append& a) {
    if (per_seq) {   // so many places a sequence
        b = item / per_seq;
        i = item - b * per_seq;
        a = append(p, b);
        return i < append_blocks(a);
    }
    for (int base = 0, before = 0; base < p.B; base += 64) {
        const int s = base + (threadIdx.x & 63);
        const int mine = s < p.B ? append_blocks(append(p, s)) : 0, upto = before + wave_sums(mine);
        const uint64_t who = __ballot(item < upto);
        if (who) {
            const int l = __builtin_ctzll(who);
            b = base + l;
            i = item - __builtin_amdgcn_readlane(upto - mine, l);
            a = append(p, b);
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// how a key is rotated: pairs of dimensions i and i + rot / 2 (EIGHTS: rot / 2 is a multiple of eight, partners are read eight
// by eight), or 2 i and 2 i + 1
enum Turn { NONE, HALVES, EIGHTS, PAIRED };

// The position of the row of token t in its sequence, rows cu_q[b] .. cu_q[b + 1] - 1 (without cu_q: row b) of which end at
// token kv_lens[b] - 1. false: it is of none. By a whole wave: each step tells 64 parts of the sequences apart.
__device__ __forceinline__ bool place_of(const Kv8WriteParams& p, int t, int& position) {
    if (!p.cu_q) {
        position = p.kv_lens[t] - 1;
        return true;
    }
    const int lane = threadIdx.x & 63;
    int at = 0, n = p.B + 1;   // the last of cu_q[at .. at + n - 1] that is t or less
    while (n > 64) {
        const int step = (n + 63) / 64, i = lane * step;
        const int k = __popcll(__ballot(i < n && p.cu_q[at + min(i, n - 1)] <= t));
        if (k == 0) return false;
        at += (k - 1) * step;
        n = min(step, n - (k - 1) * step);
    }
    const int e = min(at + lane, p.B), first = p.cu_q[e], next = p.cu_q[min(e + 1, p.B)], len = p.kv_lens[min(e, p.B - 1)];
    const int k = __popcll(__ballot(lane < n && first <= t));
    if (k == 0 || at + k > p.B) return false;
    position = __builtin_amdgcn_readlane(len, k - 1) - min(max(__builtin_amdgcn_readlane(next, k - 1), 0), p.T) + t;
    return true;
}

// Queries of one token, all heads, as rope.hip.
template <typename E, bool PAIRS, int THREADS>
__device__ __forceinline__ void turn_queries(const Kv8WriteParams& p, int D, int t, float2* turn) {
    const int half = p.rot / 2, units = row_units(p.rot, D, PAIRS), all = units * p.q.H;
    for (int e0 = 0; e0 < all; e0 += THREADS) {
        const int e = e0 + threadIdx.x, h = e / units, u = e - h * units;
        const uint16_t* x = static_cast<const uint16_t*>(p.q.x) + (size_t)t * p.q.st + (size_t)h * p.q.sh;
        uint16_t* o = static_cast<uint16_t*>(p.q.out) + (size_t)t * p.q.o_st + (size_t)h * p.q.o_sh;
        Unit v{};
        if (e < all) v = load_unit<PAIRS>(x, x == o, u, p.rot, D);
        if (e0 == 0) {   // while the first of them are on their way
            int position;
            if (p.positions) position = p.positions[t];
            else if (!place_of(p, t, position)) return;   // of no sequence: left as it is
            for (int i = threadIdx.x; i < half; i += THREADS) turn[i] = angle(position, p.inv_freq[i], p.q_magnitude.part);
            __syncthreads();
        }
        if (e < all) store_turned<E, PAIRS>(v, x == o, o, turn, p.q_magnitude.up, u, p.rot, D);
    }
}

template <typename E, int D, Turn TURN>
__global__ __launch_bounds__(2 * D) void kv8_write_kernel(Kv8WriteParams p, int per_seq, int items, int groups, int heads) {
    constexpr int ROW = D + 8, THREADS = 2 * D;
    __shared__ __align__(16) uint16_t rows[2][16][ROW];
    __shared__ uint32_t top[2][16];                     // largest magnitude of a row, as bits
    __shared__ __align__(16) float2 turn[TURN == NONE ? 1 : 16][TURN == NONE ? 1 : D / 2 + 2];   // 16 rows, each four banks on
    if ((int)blockIdx.x >= items * groups) {
        if constexpr (TURN != NONE) turn_queries<E, TURN == PAIRED, THREADS>(p, D, blockIdx.x - items * groups, &turn[0][0]);
        return;
    }
    const int item = blockIdx.x / groups, h0 = (blockIdx.x - item * groups) * heads;
    int b, i;
    Append a;
    if (!find_block(p, per_seq, item, b, i, a)) return;
    const int blk = (a.lo >> 4) + i, from = max(a.lo - 16 * blk, 0), to = min(a.hi - 16 * blk, 16);   // new tokens of the block
    const int page = p.table[(size_t)b * p.pages_per_seq + ((16 * blk) >> p.page_shift)];
    if ((unsigned)page >= (unsigned)p.num_pages) return;
    const int row0 = a.row + 16 * blk - a.lo;           // row of token 0 of the block
    const int x = threadIdx.x;
    if constexpr (TURN != NONE) {
        const int half = p.rot / 2;
        for (int e = x; e < (to - from) * half; e += THREADS) {
            const int t = from + e / half, f = e - (t - from) * half;
            turn[t][f] = angle(p.positions ? p.positions[row0 + t] : 16 * blk + t, p.inv_freq[f], p.magnitude);
        }
    }
    const bool values = x >= D;
    const int y = values ? x - D : x;
    for (int h = h0; h < min(h0 + heads, p.Hkv); ++h) {
        unsigned char* block = p.cache + (((((size_t)page * p.Hkv + h) << (p.page_shift - 4)) + (blk & ((1 << (p.page_shift - 4)) - 1))) * kv8_block_bytes(D));
        const u32x4 tail = *reinterpret_cast<const u32x4*>(block + 32 * D);
        // rows into LDS: eight elements of either matrix, then eight more
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int e = y + r * D, t = e / (D / 8), d = 8 * (e - t * (D / 8));
            if (t >= from && t < to) {
                const uint16_t* src = values ? static_cast<const uint16_t*>(p.v) + (size_t)(row0 + t) * p.v_st + (size_t)h * p.v_sh
                                             : static_cast<const uint16_t*>(p.k) + (size_t)(row0 + t) * p.k_st + (size_t)h * p.k_sh;
                *reinterpret_cast<u32x4*>(&rows[values][t][d]) = *reinterpret_cast<const u32x4*>(src + d);
            }
        }
        if (x < 32) top[x >> 4][x & 15] = 0;
        __syncthreads();
        // this thread's 16 values: of keys dimensions 16 (y / 16).. of token y % 16; of values token 4 quad + i, dimension e
        float f[16];
        const int quad = (y >> 4) & 3, g = y >> 6, r = y & 15;
        if (!values) {
            const int t = y & 15, c = 16 * (y >> 4);
            const uint16_t* src = rows[0][t];
            uint32_t most = 0;
            if (t >= from && t < to) {
#pragma unroll
                for (int e = 0; e < 16; ++e) f[e] = elem_to_f32<E>(src[c + e]);
                const int half = p.rot / 2;
                if constexpr (TURN == EIGHTS) {
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const int d = c + 8 * g;
                        if (d < p.rot) {
                            const bool low = d < half;
                            const int i = low ? d : d - half;
                            float other[8];
                            to_f32<E>(*reinterpret_cast<const Elems8*>(src + (low ? d + half : i)), other);
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                float u = low ? f[8 * g + e] : other[e], w = low ? other[e] : f[8 * g + e];
                                turn_pair(u, w, turn[t][i + e]);
                                f[8 * g + e] = low ? u : w;
                            }
                        }
                    }
                } else if constexpr (TURN == HALVES) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int d = c + e;
                        if (d < p.rot) {
                            const bool low = d < half;
                            const float other = elem_to_f32<E>(src[low ? d + half : d - half]);
                            float u = low ? f[e] : other, v = low ? other : f[e];
                            turn_pair(u, v, turn[t][low ? d : d - half]);
                            f[e] = low ? u : v;
                        }
                    }
                } else if constexpr (TURN == PAIRED) {
#pragma unroll
                    for (int e = 0; e < 16; e += 2)
                        if (c + e < p.rot) turn_pair(f[e], f[e + 1], turn[t][(c + e) >> 1]);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) most = max(most, __float_as_uint(f[e]) & 0x7FFFFFFFu);
                atomicMax(&top[0][t], most);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = 4 * quad + i;
                if (t >= from && t < to) {
                    const u32x2 w = *reinterpret_cast<const u32x2*>(&rows[1][t][r * (D / 16) + 4 * g]);
                    uint32_t most = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        f[4 * i + e] = elem_to_f32<E>(w[e >> 1] >> (16 * (e & 1)));
                        most = max(most, __float_as_uint(f[4 * i + e]) & 0x7FFFFFFFu);
                    }
                    most = row_max(most);
                    if (r == 0) atomicMax(&top[1][t], most);
                }
            }
        }
        __syncthreads();
        // largest finite row, and rows that are not (16 lanes have a row each, the wave's others the same)
        const uint32_t theirs = top[values][x & 15], odd = (uint32_t)__ballot(theirs >= 0x7F800000u) & 0xFFFFu;
        const uint32_t most = row_max(theirs >= 0x7F800000u ? 0u : theirs);
        // most <= 448 2^e: 448 is 1.75 2^8
        int e2 = max((int)(most >> 23) - 127 - 8 + ((most & 0x7FFFFFu) > 0x600000u ? 1 : 0), KV8_LEAST_EXP);
        const float need = pow2(e2), old = __uint_as_float(values ? tail[1] : tail[0]);
        const float s = from > 0 ? fmaxf(need, old) : need, by = 1.f / s, ratio = old * by;
        const bool shrink = from > 0 && old < s;   // the older rows' bytes are taken down
        unsigned char* const at = block + (values ? 16 * D : 0) + 16 * y;
        if (!values) {
            const int t = y & 15;
            if (t >= from && t < to) {
                const bool zero = (odd >> t) & 1;
                u32x4 w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = zero ? 0u : to_e4m3(f[4 * i] * by, f[4 * i + 1] * by, f[4 * i + 2] * by, f[4 * i + 3] * by);
                *reinterpret_cast<u32x4*>(at) = w;
            } else if (t < from && shrink) {
                u32x4 w = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = rescale(w[i], ratio);
                *reinterpret_cast<u32x4*>(at) = w;
            }
        } else if ((4 * quad + 3 >= from && 4 * quad < to) || (4 * quad < from && shrink)) {
            uint32_t fresh = 0, older = 0;   // bytes of new rows, of older ones
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = 4 * quad + i;
                if (t >= from && t < to) {
                    fresh |= 255u << (8 * i);
                    if ((odd >> t) & 1)
#pragma unroll
                        for (int e = 0; e < 4; ++e) f[4 * i + e] = 0.f;
                } else {
                    if (t < from) older |= 255u << (8 * i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) f[4 * i + e] = 0.f;
                }
            }
            u32x4 w = {0, 0, 0, 0};
            if (fresh != ~0u) w = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t kept = w[e];
                if (shrink) kept = (kept & ~older) | (rescale(kept, ratio) & older);
                w[e] = (kept & ~fresh) | (to_e4m3(f[e] * by, f[4 + e] * by, f[8 + e] * by, f[12 + e] * by) & fresh);
            }
            *reinterpret_cast<u32x4*>(at) = w;
        }
        // scales and rows that are not finite: the keys' by one thread, the values' by another
        if (y == 0) {
            const uint32_t before = (1u << from) - 1u;
            reinterpret_cast<float*>(block + 32 * D)[values] = s;
            reinterpret_cast<uint16_t*>(block + 32 * D + 8)[values] = (uint16_t)(((tail[2] >> (values ? 16 : 0)) & before) | odd);
            if (values) reinterpret_cast<uint32_t*>(block + 32 * D)[3] = 0;
        }
        __syncthreads();
    }
}

template <typename E, int D>
__global__ __launch_bounds__(256) void kv8_read_kernel(Kv8ReadParams p) {
    constexpr int N = D / 16;   // a lane's elements of a row
    const int r = threadIdx.x & 15, t = blockIdx.x * 16 + (threadIdx.x >> 4), h = blockIdx.y;
    if (t >= p.T) return;
    const int slot = p.slots[t], page = slot >> p.page_shift;
    if (slot < 0 || page >= p.num_pages) return;
    const int in_page = slot & ((1 << p.page_shift) - 1), tok = in_page & 15;
    const unsigned char* block = p.cache + ((((size_t)page * p.Hkv + h) << (p.page_shift - 4)) + (in_page >> 4)) * kv8_block_bytes(D);
    const u32x4 tail = *reinterpret_cast<const u32x4*>(block + 32 * D);
    uint32_t k[N / 4], v[N / 4][4];
#pragma unroll
    for (int x = 0; x < N / 4; ++x) {
        const int d = r * N + 4 * x;
        k[x] = *reinterpret_cast<const uint32_t*>(block + (d >> 4) * 256 + 16 * tok + (d & 15));
        const u32x4 u = *reinterpret_cast<const u32x4*>(block + 16 * D + 1024 * x + (tok >> 2) * 256 + 16 * r);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[x][e] = u[e] >> (8 * (tok & 3));
    }
    const float sk = (tail[2] >> tok) & 1 ? __builtin_nanf("") : __uint_as_float(tail[0]);
    const float sv = (tail[2] >> (16 + tok)) & 1 ? __builtin_nanf("") : __uint_as_float(tail[1]);
    uint16_t* ok = static_cast<uint16_t*>(p.k_out) + (size_t)t * p.k_st + (size_t)h * p.k_sh + r * N;
    uint16_t* ov = static_cast<uint16_t*>(p.v_out) + (size_t)t * p.v_st + (size_t)h * p.v_sh + r * N;
#pragma unroll
    for (int x = 0; x < N / 4; ++x) {
        float f[4], g[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[e] = saturate<E>(byte_f32(k[x], e) * sk);
            g[e] = saturate<E>(byte_f32(v[x][e], 0) * sv);
        }
        *reinterpret_cast<u32x2*>(ok + 4 * x) = u32x2{pack2(E{}, f[0], f[1]), pack2(E{}, f[2], f[3])};
        *reinterpret_cast<u32x2*>(ov + 4 * x) = u32x2{pack2(E{}, g[0], g[1]), pack2(E{}, g[2], g[3])};
    }
}

template <typename E, int D>
static void write(const Kv8WriteParams& p, hipStream_t st) {
    // blocks that max_q tokens in a row may lie in, and that all of them may: whichever gives fewer places
    const long long per = ((long long)(p.max_q < p.T ? p.max_q : p.T) + 30) / 16, all = (long long)p.T / 16 + 2 * (long long)p.B;
    const bool direct = per * p.B <= 2 * all;
    const int items = (int)(direct ? per * p.B : all);
    // Heads of a workgroup: more share a token's angles, fewer fill the device, so twice as many as long as 2048 places for workgroups
    // are left; 1024 beside queries, whose workgroups fill it, too. (Places: with max_q_len given, of sequences of all lengths, up to half of
    // them are empty.) 8 heads of D = 128, us for 1, 2, 4, 8 a workgroup (captured, the same rows each time), * what the rule takes: 5 prompts
    // of 60 to 2048 tokens with 32 heads of queries 31.6, 27.7, 24.8*, 26.8, without max_q_len 32.7, 28.2*, 25.5, 25.4, keys alone 19.9,
    // 17.6*, 18.9, 24.5; 8192 tokens 43.6, 37.7, 34.5*, 35.2 and 25.5, 20.0*, 18.2, 23.2; 64 sequences of 64 25.4, 23.4*, 21.2, 24.4
    // and 15.2*, 12.0, 14.8, 20.5; 2048 tokens 14.4*, 13.7, 14.7, 23.2 and 9.0*, 9.0, 12.0, 19.5.
    int heads = 1;
    while (heads < p.Hkv && (long long)items * ((p.Hkv + 2 * heads - 1) / (2 * heads)) >= (p.q.H ? 1024 : 2048)) heads *= 2;
    const int groups = (p.Hkv + heads - 1) / heads;
    const unsigned grid = (unsigned)items * groups + (p.q.H ? p.T : 0);
    const int per_seq = direct ? (int)per : 0;
    if (!p.inv_freq) kv8_write_kernel<E, D, NONE><<<grid, 2 * D, 0, st>>>(p, per_seq, items, groups, heads);
    else if (p.interleaved) kv8_write_kernel<E, D, PAIRED><<<grid, 2 * D, 0, st>>>(p, per_seq, items, groups, heads);
    else if (p.rot % 16 == 0) kv8_write_kernel<E, D, EIGHTS><<<grid, 2 * D, 0, st>>>(p, per_seq, items, groups, heads);
    else kv8_write_kernel<E, D, HALVES><<<grid, 2 * D, 0, st>>>(p, per_seq, items, groups, heads);
}
template <typename E, int D>
static void read(const Kv8ReadParams& p, hipStream_t st) { kv8_read_kernel<E, D><<<dim3((p.T + 15) / 16, p.Hkv), 256, 0, st>>>(p); }

hipError_t launch_kv8_write(bool bf16, int D, const Kv8WriteParams& p, hipStream_t st) {
    switch (D) {
        case 64: bf16 ? write<bf16_t, 64>(p, st) : write<half_t, 64>(p, st); break;
        case 128: bf16 ? write<bf16_t, 128>(p, st) : write<half_t, 128>(p, st); break;
        case 192: bf16 ? write<bf16_t, 192>(p, st) : write<half_t, 192>(p, st); break;
        case 256: bf16 ? write<bf16_t, 256>(p, st) : write<half_t, 256>(p, st); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}
hipError_t launch_kv8_read(bool bf16, int D, const Kv8ReadParams& p, hipStream_t st) {
    switch (D) {
        case 64: bf16 ? read<bf16_t, 64>(p, st) : read<half_t, 64>(p, st); break;
        case 128: bf16 ? read<bf16_t, 128>(p, st) : read<half_t, 128>(p, st); break;
        case 192: bf16 ? read<bf16_t, 192>(p, st) : read<half_t, 192>(p, st); break;
        case 256: bf16 ? read<bf16_t, 256>(p, st) : read<half_t, 256>(p, st); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace w4a16
