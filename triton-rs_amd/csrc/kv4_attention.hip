// Attention over the 4-bit key/value cache (kv4.h).
//
// Query row i of sequence b stands at position kv_len - q_len + i and sees key j < kv_len where
// (causal) j <= its position and (window) j > its position - window:
//   w_j = scale q . k_j,  out = sum_j exp(w_j - m) v_j / sum_j exp(w_j - m),  lse = m + ln sum
// in one pass over the keys with a running m. No visible key: out = 0, lse = -infinity.
// One wave a query row and head.
#include "device_common.h"
#include "kv4.h"

namespace w4a16 {

template <typename E>
__device__ __forceinline__ float param_scale(uint32_t w) {
    if constexpr (__is_same(E, half_t)) return (float)__builtin_bit_cast(half_t, (uint16_t)w);
    else return bf16_bits_to_f32(w & 0xFFFFu);
}

template <typename E, int D>
__global__ __launch_bounds__(64) void kv4_attention_kernel(Kv4AttnParams p) {
    __shared__ float qs[D];
    __shared__ float ps[16];
    const int lane = threadIdx.x, b = blockIdx.y, a = blockIdx.z, i = blockIdx.x;
    const int q0 = p.cu_q ? min(max(p.cu_q[b], 0), p.T) : b;
    const int q1 = p.cu_q ? min(max(p.cu_q[b + 1], 0), p.T) : b + 1;
    const int n = q1 - q0;
    if (i >= n) return;
    const int t = q0 + i, h = a / (p.Hq / p.Hkv);
    const long long cap = (long long)p.pages_per_seq << p.page_shift;
    const int len = (int)min((long long)min(p.kv_lens[b], p.max_kv), cap);
    const int pos = len - n + i;
    const int hi = p.causal ? min(len, pos + 1) : len;
    const int lo = p.window ? max(0, pos - p.window + 1) : 0;
    const E* q = static_cast<const E*>(p.q) + (size_t)t * p.q_st + (size_t)a * p.q_sh;
    for (int d = lane; d < D; d += 64) qs[d] = (float)q[d];
    __syncthreads();
    constexpr int N = D / 64;
    float o[N] = {}, m = -INFINITY, l = 0.f;
    const int tok = lane & 15, part = lane >> 4;
    for (int j0 = lo & ~15; j0 < hi; j0 += 16) {
        const int page = p.table[(size_t)b * p.pages_per_seq + (j0 >> p.page_shift)];
        if (page < 0 || page >= p.num_pages) continue;
        const unsigned char* block = p.cache +
            (((size_t)page * p.Hkv + h) * (1 << (p.page_shift - 4)) + ((j0 & ((1 << p.page_shift) - 1)) >> 4)) * kv4_block_bytes(D);
        const uint32_t* kw = reinterpret_cast<const uint32_t*>(block + tok * (D / 2) + part * (D / 8));
        const uint32_t par = reinterpret_cast<const uint32_t*>(block + 16 * D)[tok];
        float dot = 0.f;
        for (int w = 0; w < D / 32; ++w)
            for (int e = 0; e < 8; ++e)
                dot += qs[part * (D / 4) + 8 * w + e] * ((float)((kw[w] >> (4 * e)) & 15u) - (float)(par >> 16));
        dot += __shfl_xor(dot, 16);
        dot += __shfl_xor(dot, 32);
        const int j = j0 + tok;
        const bool see = j >= lo && j < hi;
        const float w = see ? dot * param_scale<E>(par) * p.scale_log2 : -INFINITY;
        float top = w;
        for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float mn = fmaxf(m, top);
        // (a row of -infinity keeps its sums at 0; NaN goes through p)
        const float base = mn == -INFINITY ? 0.f : mn, fall = exp2f(m - base);
        const float pj = see ? exp2f(w - base) : 0.f;
        float sum = pj;
        for (int x = 1; x < 16; x <<= 1) sum += __shfl_xor(sum, x);
        l = l * fall + sum;
        m = mn;
        __syncthreads();
        if (lane < 16) ps[tok] = pj;
        __syncthreads();
        for (int x = 0; x < N; ++x) {
            const int d = lane * N + x, col = d / (D / 16), r = d % (D / 16);
            float acc = o[x] * fall;
            for (int k = 0; k < 16; ++k) {
                if (j0 + k < lo || j0 + k >= hi) continue;
                const uint16_t n4 = *reinterpret_cast<const uint16_t*>(
                    block + 8 * D + (k >> 2) * (2 * D) + col * (D / 8) + ((k >> 1) & 1) * (D / 16) + (r >> 2) * 4 + 2 * (k & 1));
                const uint32_t pv = reinterpret_cast<const uint32_t*>(block + 16 * D + 64)[k];
                acc += ps[k] * ((float)((n4 >> (4 * (r & 3))) & 15) - (float)(pv >> 16)) * param_scale<E>(pv);
            }
            o[x] = acc;
        }
    }
    E* out = static_cast<E*>(p.out) + (size_t)t * p.o_st + (size_t)a * p.o_sh;
    for (int x = 0; x < N; ++x) out[lane * N + x] = (E)(l == 0.f ? 0.f : o[x] / l);
    if (p.lse && lane == 0) p.lse[(size_t)t * p.Hq + a] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

template <typename E>
static void go(int D, dim3 grid, const Kv4AttnParams& p, hipStream_t st) {
    switch (D) {
        case 64: kv4_attention_kernel<E, 64><<<grid, 64, 0, st>>>(p); break;
        case 128: kv4_attention_kernel<E, 128><<<grid, 64, 0, st>>>(p); break;
        case 192: kv4_attention_kernel<E, 192><<<grid, 64, 0, st>>>(p); break;
        default: kv4_attention_kernel<E, 256><<<grid, 64, 0, st>>>(p); break;
    }
}

hipError_t launch_kv4_attention(bool bf16, int D, const Kv4AttnParams& p, hipStream_t st) {
    const dim3 grid(p.max_q, p.B, p.Hq);
    if (bf16) go<bf16_t>(D, grid, p, st);
    else go<half_t>(D, grid, p, st);
    return hipGetLastError();
}

}  // namespace w4a16
