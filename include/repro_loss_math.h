#pragma once
// What defines the reproducible cross entropy of a vocabulary projection: the exponential, the
// logarithm and the order of every sum, callable from host and device code. Every operation is rounded
// once (build without -ffast-math and without FP contraction; fused multiply-adds are written out).
#include "repro_gemm_math.h"

namespace repro_loss {

using repro_gemm::bits_to_float;

// e^x for x <= 0, within 1.04 units in the last place; 0 below -87, where results leave the normal range; NaN
// for NaN. x = n ln 2 + r with |r| <= ln 2 / 2 (ln 2 in two parts, the first short enough for n times it to be
// exact: Cody and Waite's reduction), and Taylor's polynomial to r^7 / 7!, whose remainder is under
// 2^-27 of the result. It never falls as x rises (checked for every float32): the largest of a row's
// values is that of its largest x.
RG_HD inline float exp_in_range(float x) {
    const float n = __builtin_rintf(x * 1.44269504f);
    float r = __builtin_fmaf(n, -0.693145751953125f, x);   // 0x1.62e4p-1
    r = __builtin_fmaf(n, -1.42860677e-6f, r);             // ln 2 - 0x1.62e4p-1
    float p = 1.0f / 5040.0f;
    p = __builtin_fmaf(p, r, 1.0f / 720.0f);
    p = __builtin_fmaf(p, r, 1.0f / 120.0f);
    p = __builtin_fmaf(p, r, 1.0f / 24.0f);
    p = __builtin_fmaf(p, r, 1.0f / 6.0f);
    p = __builtin_fmaf(p, r, 0.5f);
    p = 1.0f + __builtin_fmaf(r * r, p, r);
    return bits_to_float(repro_gemm::float_to_bits(p) + ((uint32_t)(int)n << 23));  // p 2^n: p is about 0.7 to 1.42
}

RG_HD inline float exp_nonpositive(float x) { return x >= -87.0f ? exp_in_range(x) : x == x ? 0.0f : x; }

// One word's share of dz (the target's is elsewhere): 0 in a row whose factor is 0, whatever its logits.
RG_HD inline float dz_of(float z, float top, float factor) {
    const float x = z - top;
    return x >= -87.0f && factor != 0.0f ? exp_in_range(x) * factor : 0.0f;
}

// ln s in binary64 for a positive normal float32, NaN or infinity (returned as they are): s = 2^e m with m in
// [sqrt(1/2), sqrt 2), ln m = 2 artanh((m - 1) / (m + 1)) by its series to the 25th power.
RG_HD inline double log_positive(float s) {
    if (!(s < 3.4028235e38f)) return (double)s;
    const uint32_t b = repro_gemm::float_to_bits(s);
    int e = (int)(b >> 23) - 127;
    double m = (double)bits_to_float((b & 0x7FFFFFu) | 0x3F800000u);
    if (m > 1.4142135623730951) {
        m = m * 0.5;
        e += 1;
    }
    const double t = (m - 1.0) / (m + 1.0), q = t * t;
    double p = 1.0 / 25.0;
    for (int k = 23; k > 0; k -= 2) p = p * q + 1.0 / (double)k;
    return (double)e * 0.69314718055994531 + 2.0 * (t * p);
}

// ---- sums ----
//
// A token's logits z are taken in parts of PART consecutive words (the last may be shorter). A part has its
// largest logit a and its sum b of e^(z - a): chunks of 4 consecutive words (missing ones 0) give
// (v0 + v1) + (v2 + v3), and the chunks are added as a balanced tree whose first level adds chunks c and
// c + 8, the next c and c + 4, and so on; b is 0 where a is -infinity. The token's largest logit is m = max a, and its sum s that of
// b e^(a - m): part p goes to strand p mod 64, in ascending order from +0, and the strands are added as a
// balanced tree whose first level adds l and l + 32, the next l and l + 16, and so on.
constexpr int PART = 64;

// The losses' sum is taken in binary64: token n to strand n mod STRANDS, in ascending order from +0, and the
// strands as a balanced tree whose first level adds l and l + STRANDS / 2, and so on; a mean is divided by the
// count there, and either is rounded to float32 once.
constexpr int STRANDS = 1024;

// Tokens are taken in groups of this many, whose logits are held together (at most 2^27 of them,
// 512 MB, past 128 tokens). It is part of the result: a group's contribution to the weight's gradient
// is rounded once, and the groups' are added in ascending order.
constexpr int MAX_GROUP = 2048;
inline int group_tokens(long long V) {
    int r = MAX_GROUP;
    while (r > 128 && r * V > (1ll << 27)) r /= 2;
    return r;
}

// One token: what its logits' gradient is made of. `weight` is the loss's factor. Where `factor` is 0, so is the
// token's row of dz, and its row of x counts as zeros in the product for dw: what it holds (padding may hold
// anything) does not set the scale that the other tokens' values are rounded at.
struct Token {
    float top, factor;  // dz_v = e^(z_v - top) * factor for the words that are not the target
    float target;       // dz of the target word: weight * (its probability - 1)
    float loss;
};

// Where the largest logit or the loss's factor is not finite, the token's row of dz is 0 (factor 0) and its target
// word's share NaN, so that its row of dx and the target's row of dw are.
RG_HD inline Token finish_token(float m, float s, float zt, float weight) {
    Token t;
    t.top = m;
    t.factor = weight / s;
    t.target = exp_nonpositive(zt - m) * t.factor - weight;
    if (!(__builtin_fabsf(t.factor) < 3.4028235e38f) || !(__builtin_fabsf(m) < 3.4028235e38f)) {
        t.factor = 0.0f;
        t.target = __builtin_nanf("");
    }
    t.loss = (float)(((double)m - (double)zt) + log_positive(s));
    return t;
}
// Of a token whose row of x holds a NaN or an infinity, and of every token where the weight holds one (the products'
// fixed-point numbers stand for neither, so the logits may look ordinary): the same, and a NaN loss.
RG_HD inline Token broken_token() { return Token{0.0f, 0.0f, __builtin_nanf(""), __builtin_nanf("")}; }
RG_HD inline bool finite_bits(float x) { return (repro_gemm::float_to_bits(x) & 0x7F800000u) != 0x7F800000u; }
// Of a token that is left out: no gradient, no loss.
RG_HD inline Token ignored_token() { return Token{0.0f, 0.0f, 0.0f, 0.0f}; }

}  // namespace repro_loss
