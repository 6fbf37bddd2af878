// Attention over a paged cache for few columns: which keys a workgroup takes, and the join of what the
// workgroups of one sequence and head have. For kv4_few.hip and kv8_few.hip.
#pragma once
#include "kv_attn_body.h"

namespace w4a16 {

constexpr int STEP = 32;   // keys of a step

__device__ __forceinline__ unsigned wave_sum(int v) { return (unsigned)__builtin_amdgcn_readlane(wave_sums(v), 63); }
__device__ __forceinline__ int wave_max(int v) { return __builtin_amdgcn_readlane(wave_scan(v, [](int a, int b) { return max(a, b); }), 63); }

// Chunks of `steps` steps of keys in chunks of c 128 (4 c steps); -1: no columns here. Up to `whole` keys (512) stay whole, as a
// chunk more costs its partial results' way to the last one and back: one sequence, 8 heads of D = 128, 500 keys in 4 bits 9.0 us
// whole, 9.8 in chunks, 700 keys 11.0, 9.4; 4 drafts of 5 tokens, 8 heads a group, 500 keys 19.8, 20.5, 700 23.5, 17.2.
__device__ __forceinline__ int few_chunks(int steps, int c, int whole) {
    return steps < 0 ? 0 : steps <= max(whole / STEP, 4 * c) ? 1 : (steps + 4 * c - 1) / (4 * c);
}

// The length of chunks, in 128 keys, for sequences of `sum` steps together and `most` at most, total(c) their number:
// at most p.budget of them, whatever the lengths. Keys / budget or keys / (budget - B / 2) where that is enough, else
// keys / (budget - B) (the budget is twice B or more); or all sequences whole where that is estimated to take no longer.
template <typename F>
__device__ __forceinline__ int few_length(const KvAttnParams& p, unsigned sum, int most, F total) {
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
    // In steps of a full device: a round of workgroups costs p.round_cost besides its steps, a step of one workgroup alone
    // p.step_alone, joining p.join_cost. (In 4 bits 6, 0.45 and 7 of 0.85 us, measured at D = 128. Whole and in two, 8 heads: 128
    // sequences of 1000 keys 34, 49 us, 256 of 900 58, 103; 48 of 4096 56, 54. In 8 bits 3, 0.6 and 8 of 0.41 us.)
    auto cost = [&](unsigned chunks, int steps) {
        const float rounds = (float)((chunks + p.at_once - 1) / p.at_once);
        return p.round_cost * rounds + fmaxf(p.step_alone * rounds * (float)steps, (float)sum / (float)p.at_once);
    };
    if (__builtin_amdgcn_readfirstlane(cost(p.B, most) <= cost(n, min(4 * c, most)) + p.join_cost)) c = max(c, (most + 3) / 4);
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
__device__ __forceinline__ bool few_item(const KvAttnParams& p, int tile, int u, bool by_seq, KvItem& w, FewFind& find) {
    w.h = blockIdx.x;
    int lo = 0, hi = 0;
    if (p.whole) {   // sequence u, in one chunk
        w.sequence<WG_COLS, STEP>(p, u, tile * WG_COLS, lo, hi);
        w.take(0, 1, 0, lo, hi);
        w.at = w.slot = 0;   // (no partial results)
        return w.cols > 0;
    }
    KvItem mine;
    auto look = [&](int b) {   // steps of sequence b, -1 without columns
        mine.sequence<WG_COLS, STEP>(p, min(b, p.B - 1), tile * WG_COLS, lo, hi);
        return b < p.B && mine.cols > 0 ? (hi - lo + STEP - 1) / STEP : -1;
    };
    int at, chunks, c;
    if (p.B <= 64) {
        const int lane = threadIdx.x & 63, steps = look(lane);
        c = few_length(p, wave_sum(max(steps, 0)), wave_max(max(steps, 0)), [&](int c) { return wave_sum(few_chunks(steps, c, p.whole_keys)); });
        const int here = few_chunks(steps, c, p.whole_keys), upto = wave_sums(here);
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
            each([&](int, int steps) { n += few_chunks(steps, c, p.whole_keys); });
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
                const unsigned here = few_chunks(steps, c, p.whole_keys);
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

// Joins the chunks of one sequence and head where that is more than one workgroup does in passing: 64 quads of
// values a workgroup, a quarter of the chunks a wave.
struct FewJoin {
    float4_t vals[256];
    float ml[256][2];
    FewFind find;
};
template <typename E, int D, int NT, int DOWN>
__device__ __forceinline__ void few_join(const KvAttnParams& p, FewJoin& lds) {
    constexpr int COLS = 32 * NT;
    KvItem w;
    const int tile = p.tiles == 1 ? 0 : blockIdx.z / p.join_parts;
    if (!few_item<COLS>(p, tile, blockIdx.y, true, w, lds.find) || w.chunks == 1) return;
    const KvSink<E, D, DOWN> sink(p, w);
    const int e = (blockIdx.z - tile * p.join_parts) * 64 + (threadIdx.x & 63);
    sink.join_quads(e, threadIdx.x >> 6, 4, 64, e < w.cols * (D / 4), lds.vals, lds.ml);
}

}  // namespace w4a16
