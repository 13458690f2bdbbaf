#pragma once
// Scalar arithmetic that defines the reproducible AdamW step, callable from host and device code:
// additions, multiplications, one division and one square root per value, each rounded once to
// float32 in a fixed order (build without -ffast-math and without FP contraction), and the 8-bit
// form of the two moments. So a step gives the same bits on every device.
#include "repro_gemm_math.h"

namespace repro_adamw {

using repro_gemm::bits_to_float;
using repro_gemm::float_to_bits;

// A step's constants, each computed in binary64 and rounded once to float32.
struct Scalars {
    float keep;          // 1 - lr * weight_decay
    float b1, c1;        // beta1, 1 - beta1
    float b2, c2;        // beta2, 1 - beta2
    float inverse, eps;  // 1 / sqrt(1 - beta2^step)
    float step;          // lr / (1 - beta1^step)
    uint32_t salt;       // of the 8-bit moments' rounding
};

inline double whole_power(double b, long long n) {
    double r = 1.0;
    for (; n > 0; n >>= 1, b *= b)
        if (n & 1) r *= b;
    return r;
}

inline Scalars make_scalars(double lr, double beta1, double beta2, double eps, double weight_decay,
                            long long step) {
    Scalars s;
    s.keep = (float)(1.0 - lr * weight_decay);
    s.b1 = (float)beta1;
    s.c1 = (float)(1.0 - beta1);
    s.b2 = (float)beta2;
    s.c2 = (float)(1.0 - beta2);
    s.inverse = (float)(1.0 / std::sqrt(1.0 - whole_power(beta2, step)));
    s.eps = (float)eps;
    s.step = (float)(lr / (1.0 - whole_power(beta1, step)));
    s.salt = (uint32_t)step * 0x9E3779B9u;  // 2^32 over the golden ratio
    return s;
}

// One value's step: m and v are replaced, the new parameter is returned.
RG_HD inline float update(float p, float g, float& m, float& v, const Scalars& s) {
    m = m * s.b1 + g * s.c1;
    v = v * s.b2 + (g * g) * s.c2;
    const float root = __builtin_sqrtf(v) * s.inverse + s.eps;
    return p * s.keep - m / root * s.step;
}

// ---- moments in 8 bits ----
//
// BLOCK consecutive values of a tensor share the float32 exponent field e of their largest
// magnitude (at least span + 4), one more where that magnitude is past the codes of its binade, 1.875
// times its power of two (cut off there, a moment that grows slowly would never pass it). With k = max(exponent field of a, e - span), a magnitude a is
// q * 2^(k - 130) for a q < 16, rounded to a whole number, and its code is 8 (k - (e - span)) + q:
// three significant bits below the leading one over span binades, equally spaced below them. The
// first moment takes a sign bit and 14 binades, the second, which is not negative, 30: as it holds
// squares, that is the same range.
// Rounding: up where the fraction of q exceeds a number in [0, 1) that mixes the value's position
// with the step, else down. To nearest, a moment that changes by less than half a code a step (one
// part in 1000 with beta2 = 0.999, against codes one part in 8 to 16 apart) would never change;
// so its expectation follows the update. A positive second moment never becomes zero: its root
// divides the step.
constexpr int BLOCK = 256;
constexpr int SPAN_M = 14, SPAN_V = 30;

RG_HD inline uint32_t mix(uint32_t h) {
    h = (h ^ (h >> 16)) * 0x6A09E667u;  // the fractions of sqrt(2) and sqrt(3)
    h = (h ^ (h >> 15)) * 0xBB67AE85u;
    return h ^ (h >> 16);
}

// The rounding numbers of the value at `position` (counted over the call's tensors, each starting at
// a whole block), 16 bits for each moment, the first one's the lower.
RG_HD inline uint32_t rounding(uint32_t position, uint32_t salt) { return mix(position ^ salt); }

// Magnitude whose exponent a block shares; infinities and NaN count as the largest finite number.
RG_HD inline uint32_t magnitude_bits(float x) {
    const uint32_t a = float_to_bits(x) & 0x7FFFFFFFu;
    return a < 0x7F7FFFFFu ? a : 0x7F7FFFFFu;
}
RG_HD inline int shared_exponent(uint32_t largest_bits, int span) {
    int e = (int)((largest_bits + (1u << 20)) >> 23);
    e = e < 254 ? e : 254;
    return e > span + 4 ? e : span + 4;
}

// The code of a magnitude, for a rounding number u16 / 65536. From 2^(e - span) on a code is the magnitude's
// exponent and upper three mantissa bits, so rounding is an addition to the float's bits whose carry
// goes where it should: 2^20 - 1 - 16 u16 carries where the lower 20 bits exceed 16 u16. Below, the
// magnitude is counted in steps of 2^(e - span - 130).
RG_HD inline int encode_magnitude(uint32_t bits, int e, int span, uint32_t u16, bool keep_positive) {
    const int low = e - span;  // an exponent field of at least 4
    const int large = (int)((bits + 0xFFFFFu - (u16 << 4)) >> 20) - 8 * (low - 1);
    const float t = bits_to_float(bits) * bits_to_float((uint32_t)(257 - low) << 23);  // exact where below 8
    const float whole = __builtin_floorf(t);
    int small = (int)whole + (t - whole > (float)(int)u16 * (1.0f / 65536.0f) ? 1 : 0);
    if (keep_positive) small = bits != 0 && small == 0 ? 1 : small;
    const int code = bits < (uint32_t)low << 23 ? small : large, top = 8 * span + 15;
    return code < top ? code : top;
}

// A code's magnitude: its bits, or below 2^(e - span) those beside 2^(e - span), which is taken away.
RG_HD inline float decode_magnitude(int code, int e, int span) {
    const int low = e > span + 4 ? e - span : 4;  // (before the first step e is 0, as the codes are)
    const uint32_t large = ((uint32_t)code << 20) + ((uint32_t)(low - 1) << 23);
    const float one = bits_to_float((uint32_t)low << 23);
    return code < 8 ? bits_to_float(large + (1u << 23)) - one : bits_to_float(large);
}

RG_HD inline uint8_t encode_m(float m, int e, uint32_t u16) {
    const int c = encode_magnitude(magnitude_bits(m), e, SPAN_M, u16, false);
    return (uint8_t)(m < 0.0f ? c + 128 : c);
}
RG_HD inline float decode_m(uint8_t code, int e) {
    const float a = decode_magnitude(code & 127, e, SPAN_M);
    return code & 128 ? -a : a;
}
RG_HD inline uint8_t encode_v(float v, int e, uint32_t u16) {
    return (uint8_t)encode_magnitude(magnitude_bits(v), e, SPAN_V, u16, true);
}
RG_HD inline float decode_v(uint8_t code, int e) { return decode_magnitude(code, e, SPAN_V); }

}  // namespace repro_adamw
