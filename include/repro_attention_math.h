#pragma once
// What defines the reproducible attention and the bias of relative positions: the exponential and the order of
// every sum, callable from host and device code. Every operation is rounded once (build without -ffast-math
// and without FP contraction; fused multiply-adds are written out). Products are chains of fused
// multiply-adds in ascending order from +0, which is what the matrix cores' float32 instructions compute.
//
// Forward, for a query and a head, with c = scale log2 e (a negative scale's sign goes to the query):
//   score  s_j = fma chain over d of q_d k_jd;  with a bias t_j = fma(s_j, c, bias_j log2 e), else t_j = s_j c
//   keys are taken in chunks of CHUNK, a chunk in tiles of TILE: m' = max(m, visible t of the tile) from m = NONE, a = rescale(m, m');
//   p_j = e2(less(t_j, m')); l_even = l_even a, then + p_j of the even keys in ascending order,
//   l_odd likewise; o_d = o_d a, then the chain over the tile's keys of p_j v_jd
//   less(t_j, m') = t_j - m', without a bias and for |m'| below LARGE fma(s_j, c, -m'), which spares a multiplication and t's rounding. (m' is
//   rounded, so the largest key's own fma is up to half a unit in m's last place away from 0: at most 1/2 there, but 2^7 at 2^31.)
//   chunks are joined in ascending order: M' = max(M, m), a = rescale(M, M'), b = rescale(m, M'),
//   L = fma(l_even + l_odd, b, L a), O_d = fma(o_d, b, O_d a)
//   y_d = O_d (1 / L)
// A masked key has p = 0 and nothing else of it takes part; a tile or chunk without visible keys changes nothing. So a
// row's bits depend on its query and the keys it sees alone, not on the batch, the other queries or the padding.
// NONE as a maximum counts as 0 in the exponents; a row that sees nothing has L = 0, which 1 / L is 0 for. A NaN or infinite t, or one
// further below the maximum than float32 reaches, gives its row NaN (holding the difference back instead costs the gradients with a bias
// registers: 3530 -> 3680 us at 2 x 16 x 4096 x 4096 x 64); a bias below LOWEST (-infinity) counts as that.
// With dropout the dropped p_j are 0 in the chain over v (not in l) and y is multiplied by factor / L.
//
// Backward: p_ij = e2(less(t_ij, M_i)) (1 / L_i), delta_i = sum_d dy_d y_d, u_ij = p_ij kept factor,
//   ds_ij = p_ij ((dy_i . v_j) kept factor - delta_i)
// Queries are taken in chunks of QUERY_CHUNK and keys in blocks of KEY_BLOCK:
//   dv_j = sum over the group's heads of the sum over the chunks, both ascending, of the chunk's chain of u_ij dy_i; dk_j likewise of
//   ds_ij q_i, times scale; dq_i = sum over the key blocks of the block's chain of ds_ij k_j, times scale
//   the bias's gradient at distance j - i: over the key blocks, the batch, the chunks, ascending, the sum of ds_ij
//   of one block and chunk in ascending order of i
#include "repro_gemm_math.h"

namespace repro_attention {

using repro_gemm::bits_to_float;
using repro_gemm::float_to_bits;

constexpr int TILE = 64, CHUNK = 256, QUERY_CHUNK = 256, KEY_BLOCK = 128, MAX_D = 128;
constexpr float LOG2E = 1.44269504f, NONE = -__builtin_inff(), LOWEST = -1e30f, LARGE = 16777216.0f;
inline float score_factor(double scale) { return (float)(scale * 1.4426950408889634); }

// 2^x for finite x up to 0 and a rounding past it, within 2.73 units in the last place (most at -0.00039, just below a power of two) or 2^-22.5,
// over every float; 1 for 0, NaN for NaN and infinities. x = n + f
// with n = floor x and 0 <= f < 1 (what rounds to 1 is the number before it); 2^f by a polynomial whose coefficients were fitted
// to the least largest relative error (2^-23.3); times 2^n, rounded once where the result is subnormal.
RG_HD inline float e2(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
    int n;
    asm("v_cvt_flr_i32_f32 %0, %1" : "=v"(n) : "v"(x));
    const float f = __builtin_amdgcn_fractf(x);
#else
    const float below = __builtin_floorf(x);
    float f = x - below;
    f = f > 0.99999994f ? 0.99999994f : f;
    const int n = below < -1000.0f ? -1000 : below > 1000.0f ? 1000 : below == below ? (int)below : 0;
#endif
    float p = 0.00186713f;
    p = __builtin_fmaf(p, f, 0.009017031f);
    p = __builtin_fmaf(p, f, 0.055799913f);
    p = __builtin_fmaf(p, f, 0.24016444f);
    p = __builtin_fmaf(p, f, 0.6931513f);
    p = __builtin_fmaf(p, f, 1.0f);
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_ldexpf(p, n);
#else
    return (float)((double)p * __builtin_bit_cast(double, (uint64_t)(1023 + n) << 52));
#endif
}
RG_HD inline float base_of(float m) { return m == NONE ? 0.0f : m; }
RG_HD inline bool is_large(float base) { return !(__builtin_fabsf(base) < LARGE); }
// less(t, base), for t = s c where there is no bias.
RG_HD inline float less(float s, float t, float c, float base, bool biased) {
    return biased || is_large(base) ? t - base : __builtin_fmaf(s, c, -base);
}
RG_HD inline float bias_term(float bias) {
    const float b = bias * LOG2E;
    return b < LOWEST ? LOWEST : b;
}
// The factor for what was summed under the maximum m: 0 where nothing was, or where the two are further apart than float32 reaches.
RG_HD inline float rescale(float m, float base) {
    const float x = m - base;
    return e2(x < LOWEST ? LOWEST : x);
}
// The larger of the two; the other where one is NaN.
RG_HD inline float larger(float a, float b) { return __builtin_fmaxf(a, b); }
// 1 / L, and 0 for a row that sees nothing.
RG_HD inline float reciprocal(float total) { return total == 0.0f ? 0.0f : 1.0f / total; }
RG_HD inline float ds_of(float p, float dp, float delta) { return p * (dp - delta); }

// The sum of x_i over a row of D <= 128 values of products x_d = a_d b_d: lane l of 64 has fma(a_{l+64}, b_{l+64}, a_l b_l)
// (missing values 0), and the lanes are added as a balanced tree whose first level adds l and l + 32, the next l and l + 16.

// ---- the bias of relative positions ----
//
// The bucket of a distance n >= 0 is the number of borders <= n (ascending, made by the caller); a bidirectional table's
// keys after the query have the upper half of the buckets.
RG_HD inline int bucket_of(long long relative, const int* borders, int count, bool both) {
    const long long n = relative > 0 ? (both ? relative : 0) : -relative;
    int low = 0, high = count;
    while (low < high) {
        const int mid = (low + high) / 2;
        if (borders[mid] <= n) low = mid + 1;
        else high = mid;
    }
    return both && relative > 0 ? low + count + 1 : low;
}
// The gradient of a dense bias: rows in runs of RUN give each distance a sum in ascending order, the runs' are added in ascending
// order; a bucket's distances (column n of [H][Tq + Tk - 1] goes to strand n mod STRANDS, in ascending order) are added, and
// the strands as a balanced tree whose first level adds s and s + STRANDS / 2.
constexpr int RUN = 64, STRANDS = 256;

}  // namespace repro_attention
