// C-ABI entry points of the norm and of rotary positions: argument checks (before any HIP call), then the
// launchers of norm.hip and rope.hip.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/w4a16.h"
#include "kv_api.h"
#include "layer.h"

namespace w4a16 {

// group: -1 for a result in the element type
static int rms_norm(void* stream, int elem, const void* x, int32_t x_st, int32_t x_sh, const void* residual, int32_t r_st,
                    int32_t r_sh, void* residual_out, int32_t ro_st, int32_t ro_sh, const void* weight, void* out, int32_t o_st,
                    int32_t o_sh, float* scales, int32_t T, int32_t H, int32_t K, int32_t group, float eps) {
    if (int rc = check_elem(elem)) return rc;
    if (T < 0 || H < 1 || K < 1) return fail(W4A16_ERR_INVALID_ARG, "bad sizes (T=%d H=%d K=%d)", T, H, K);
    if (K > NORM_MAX_K) return fail(W4A16_ERR_UNSUPPORTED, "K=%d: at most %d", K, NORM_MAX_K);
    if ((int64_t)T * H > LAYER_MAX_ROWS) return fail(W4A16_ERR_UNSUPPORTED, "%d x %d rows: at most 2^30 in a call", T, H);
    if (!(eps >= 0.f) || !std::isfinite(eps)) return fail(W4A16_ERR_INVALID_ARG, "eps must be finite and not negative");
    if (group > 0 && (group < 32 || group > 512 || (group & (group - 1)) || K % group))
        return fail(W4A16_ERR_INVALID_ARG, "group %d: 0 (a row), 32, 64, 128, 256 or 512, and K=%d a multiple", group, K);
    if (T == 0) return W4A16_OK;
    if (!weight || (group >= 0 && !scales)) return fail(W4A16_ERR_INVALID_ARG, "null pointer argument (weight or scales)");
    if ((uintptr_t)weight % 2 || (uintptr_t)scales % 4) return fail(W4A16_ERR_INVALID_ARG, "weight must be 2-byte aligned, scales 4-byte");
    if (!residual != !residual_out) return fail(W4A16_ERR_INVALID_ARG, "null pointer argument (residual and residual_out: both or neither)");
    if (int rc = check_rows("x", x, x_st, x_sh, T, H, K, 1, false)) return rc;
    if (residual)
        if (int rc = check_rows("residual", residual, r_st, r_sh, T, H, K, 1, false)) return rc;
    if (residual)
        if (int rc = check_rows("residual_out", residual_out, ro_st, ro_sh, T, H, K, 1, true)) return rc;
    if (group < 0) {
        if (int rc = check_rows("out", out, o_st, o_sh, T, H, K, 1, true)) return rc;
    } else if (int rc = check_rows("out", out ? weight : nullptr, o_st, o_sh, T, H, K, 1, true)) {   // (bytes lie at any address)
        return rc;
    }
    NormParams p{};
    p.x = x; p.residual = residual; p.weight = weight; p.residual_out = residual_out; p.out = out; p.scales = scales;
    p.x_st = x_st; p.x_sh = x_sh; p.r_st = r_st; p.r_sh = r_sh; p.ro_st = ro_st; p.ro_sh = ro_sh; p.o_st = o_st; p.o_sh = o_sh;
    p.T = T; p.H = H; p.K = K; p.group = group == K ? 0 : group; p.eps = eps;
    (void)hipGetLastError();
    const hipError_t e = launch_norm(elem == W4A16_BF16, p, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? W4A16_OK : hip_fail(e, "rms_norm launch");
}

}  // namespace w4a16

using namespace w4a16;

extern "C" {

W4A16_API int w4a16_rms_norm(void* stream, int elem, const void* x, int32_t x_stride_t, int32_t x_stride_h,
                             const void* residual, int32_t r_stride_t, int32_t r_stride_h, void* residual_out,
                             int32_t ro_stride_t, int32_t ro_stride_h, const void* weight, void* out, int32_t out_stride_t,
                             int32_t out_stride_h, int32_t T, int32_t H, int32_t K, float eps) {
    return rms_norm(stream, elem, x, x_stride_t, x_stride_h, residual, r_stride_t, r_stride_h, residual_out, ro_stride_t,
                    ro_stride_h, weight, out, out_stride_t, out_stride_h, nullptr, T, H, K, -1, eps);
}

W4A16_API int w4a16_rms_norm_8bit(void* stream, int elem, const void* x, int32_t x_stride_t, int32_t x_stride_h,
                                  const void* residual, int32_t r_stride_t, int32_t r_stride_h, void* residual_out,
                                  int32_t ro_stride_t, int32_t ro_stride_h, const void* weight, void* out,
                                  int32_t out_stride_t, int32_t out_stride_h, float* scales, int32_t T, int32_t H, int32_t K,
                                  int32_t group, float eps) {
    if (group < 0) return fail(W4A16_ERR_INVALID_ARG, "group %d must not be negative", group);
    return rms_norm(stream, elem, x, x_stride_t, x_stride_h, residual, r_stride_t, r_stride_h, residual_out, ro_stride_t,
                    ro_stride_h, weight, out, out_stride_t, out_stride_h, scales, T, H, K, group, eps);
}

W4A16_API int w4a16_rope_frequencies(int32_t rot, double base, int scaling, double factor, double original_length,
                                     double slow, double fast, double* inv_freq) {
    if (rot < 2 || rot % 2 || rot > ROPE_MAX_D) return fail(W4A16_ERR_INVALID_ARG, "rot=%d: even, 2 to %d", rot, ROPE_MAX_D);
    if (!inv_freq) return fail(W4A16_ERR_INVALID_ARG, "null pointer argument (inv_freq)");
    if (!(base > 0.) || !std::isfinite(base)) return fail(W4A16_ERR_INVALID_ARG, "base must be finite and positive");
    if (scaling < W4A16_ROPE_PLAIN || scaling > W4A16_ROPE_RAMP) return fail(W4A16_ERR_INVALID_ARG, "unknown scaling %d", scaling);
    if (scaling != W4A16_ROPE_PLAIN && (!(factor > 0.) || !std::isfinite(factor)))
        return fail(W4A16_ERR_INVALID_ARG, "factor must be finite and positive");
    if (scaling == W4A16_ROPE_RAMP && (!(original_length > 0.) || !std::isfinite(original_length) || !(slow >= 0.) || !(fast > slow) || !std::isfinite(fast)))
        return fail(W4A16_ERR_INVALID_ARG, "original_length must be positive, 0 <= slow < fast");
    if (scaling == W4A16_ROPE_BASE && rot > 2) base *= std::pow(factor, (double)rot / (rot - 2));
    for (int i = 0; i < rot / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot);
        if (scaling == W4A16_ROPE_LINEAR) f /= factor;
        if (scaling == W4A16_ROPE_RAMP) {
            const double turns = original_length * f / (2.0 * 3.14159265358979323846), share = std::fmin(1.0, std::fmax(0.0, (turns - slow) / (fast - slow)));
            f *= share + (1.0 - share) / factor;
        }
        inv_freq[i] = f;
    }
    return W4A16_OK;
}

W4A16_API int w4a16_rope(void* stream, int elem, const void* q, int32_t q_stride_t, int32_t q_stride_h, void* q_out,
                         int32_t qo_stride_t, int32_t qo_stride_h, const void* k, int32_t k_stride_t, int32_t k_stride_h,
                         void* k_out, int32_t ko_stride_t, int32_t ko_stride_h, const int32_t* positions,
                         const double* inv_freq, float magnitude, int32_t T, int32_t Hq, int32_t Hkv, int32_t D, int32_t rot,
                         int32_t interleaved) {
    if (int rc = check_elem(elem)) return rc;
    if (T < 0 || Hq < 1 || Hkv < 0 || D < 1) return fail(W4A16_ERR_INVALID_ARG, "bad sizes (T=%d Hq=%d Hkv=%d D=%d)", T, Hq, Hkv, D);
    if (D > ROPE_MAX_D || Hq > KV_MAX_HEADS || Hkv > KV_MAX_HEADS)
        return fail(W4A16_ERR_UNSUPPORTED, "%d and %d heads of %d: at most %d of %d", Hq, Hkv, D, KV_MAX_HEADS, ROPE_MAX_D);
    if ((int64_t)T * (Hq > Hkv ? Hq : Hkv) > LAYER_MAX_ROWS)
        return fail(W4A16_ERR_UNSUPPORTED, "%d tokens of %d and %d rows: at most 2^30 in a call", T, Hq, Hkv);
    if (rot < 2 || rot % 2 || rot > D) return fail(W4A16_ERR_INVALID_ARG, "rot=%d: even, 2 to the head's %d dimensions", rot, D);
    if (!std::isfinite(magnitude)) return fail(W4A16_ERR_INVALID_ARG, "magnitude must be finite");
    if (!k != (Hkv == 0) || !k != !k_out) return fail(W4A16_ERR_INVALID_ARG, "k, k_out and Hkv: all or none");
    if (T == 0) return W4A16_OK;
    if (!positions || !inv_freq) return fail(W4A16_ERR_INVALID_ARG, "null pointer argument (positions or inv_freq)");
    if ((uintptr_t)positions % 4 || (uintptr_t)inv_freq % 8) return fail(W4A16_ERR_INVALID_ARG, "positions must be 4-byte aligned, inv_freq 8-byte");
    if (int rc = check_rows("q", q, q_stride_t, q_stride_h, T, Hq, D, 1, false)) return rc;
    if (int rc = check_rows("q_out", q_out, qo_stride_t, qo_stride_h, T, Hq, D, 1, true)) return rc;
    if (k) {
        if (int rc = check_rows("k", k, k_stride_t, k_stride_h, T, Hkv, D, 1, false)) return rc;
        if (int rc = check_rows("k_out", k_out, ko_stride_t, ko_stride_h, T, Hkv, D, 1, true)) return rc;
    }
    RopeParams p{};
    p.rows[0] = {q, q_out, q_stride_t, q_stride_h, qo_stride_t, qo_stride_h, Hq};
    p.rows[1] = {k, k_out, k_stride_t, k_stride_h, ko_stride_t, ko_stride_h, Hkv};
    p.positions = positions; p.inv_freq = inv_freq; p.magnitude = Magnitude::of(magnitude);
    p.T = T; p.D = D; p.rot = rot; p.interleaved = interleaved != 0;
    (void)hipGetLastError();
    const hipError_t e = launch_rope(elem == W4A16_BF16, p, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? W4A16_OK : hip_fail(e, "rope launch");
}

}  // extern "C"
