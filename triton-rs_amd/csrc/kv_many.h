// Attention over a paged cache for many columns: which tile and keys a workgroup takes, and the join of a
// tile's chunks. For kv4_many.hip and kv8_many.hip.
#pragma once
#include "kv_attn_body.h"

namespace w4a16 {

constexpr int MANY_STEP = 64;   // keys of a step

// Sequence and tile of 128 columns of this workgroup, and its chunk of the keys: those with the longest rows first, or
// (where all workgroups run at once) long and short ones by turns. p.rows: the tiles of all sequences stand in one row,
// each sequence's longest first, so that the workgroups of a prompt among single tokens lie side by side. place:
// tile and chunk, or (p.rows) chunk.
__device__ __forceinline__ bool many_tile(const KvAttnParams& p, int place, int& b, int& tile, int& chunk, size_t& at) {
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

__device__ __forceinline__ bool many_item(const KvAttnParams& p, int place, KvItem& w) {
    int b, tile, chunk, lo, hi;
    w.h = blockIdx.x;
    if (!many_tile(p, place, b, tile, chunk, w.at)) return false;
    w.sequence<128, MANY_STEP>(p, b, tile * 128, lo, hi);
    const int chunks = p.splits == 1 ? 1 : max(1, (int)(((unsigned)(hi - lo) + p.chunk - 1) / (unsigned)p.chunk));
    w.take(chunk, chunks, p.chunk, lo, hi);
    w.slot = w.at * p.splits;
    return w.cols > 0 && chunk < chunks;
}

// Joins the chunks of one tile: an eighth of its values a workgroup. (The last of the chunks' own workgroups took longer:
// 64 queries over 4096 keys, 32 heads of D = 128, 8 chunks, 40.1 us, so 30; two chunks of 400 over 2000 40.2, 39.3.)
constexpr int MANY_PARTS = 8;
template <typename E, int D, int DOWN, typename P>
__device__ __forceinline__ void many_join(const KvAttnParams& p, float* ml, P place) {   // ml: two floats a column
    KvItem w;
    const int part = blockIdx.z % MANY_PARTS;
    if (!many_item(p, blockIdx.z / MANY_PARTS * p.splits, w) || w.chunks == 1) return;   // (its results are in place)
    const KvSink<E, D, DOWN> sink(p, w);
    sink.template join_lanes<MANY_PARTS>(min(128, w.cols), ml, part, place);
}

}  // namespace w4a16
