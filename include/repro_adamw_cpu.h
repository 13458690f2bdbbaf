#pragma once
// repro_adamw_cpu.h -- the reproducible AdamW step on the host CPU (header-only C++17; no GPU
// needed), bit-identical to rg_adamw_fp32 and rg_adamw8_fp32 (include/repro_adamw.h).
//
//   cpu_adamw(p, g, m, v, n, s)                         one tensor's step
//   cpu_adamw8(p, g, m, m_exp, v, v_exp, n, first, s)   the same with the moments in 8 bits; `first`:
//                                                       the call's blocks before this tensor
//   cpu_adamw8_values(code, exp, out, blocks, signed)   what codes stand for
#include <algorithm>
#include <cstdint>

#include "repro_adamw_math.h"
#include "repro_gemm_cpu.h"

namespace repro_adamw {

inline void cpu_adamw(float* p, const float* g, float* m, float* v, int64_t n, const Scalars& s) {
    constexpr int64_t RUN = 16384;
    repro_gemm::cpu_for((int)((n + RUN - 1) / RUN), [&](int c) {
        const int64_t end = std::min(n, (c + 1) * RUN);
        for (int64_t i = c * RUN; i < end; ++i) p[i] = update(p[i], g[i], m[i], v[i], s);
    });
}

inline void cpu_adamw8(float* p, const float* g, uint8_t* m, uint8_t* m_exp, uint8_t* v, uint8_t* v_exp,
                       int64_t n, int64_t first, const Scalars& s) {
    repro_gemm::cpu_for((int)((n + BLOCK - 1) / BLOCK), [&](int b) {
        const int64_t base = (int64_t)b * BLOCK;
        const int held = (int)std::min<int64_t>(BLOCK, n - base);
        float mv[BLOCK] = {}, vv[BLOCK] = {};
        uint32_t top_m = 0, top_v = 0;
        for (int i = 0; i < held; ++i) {
            mv[i] = decode_m(m[base + i], m_exp[b]);
            vv[i] = decode_v(v[base + i], v_exp[b]);
            p[base + i] = update(p[base + i], g[base + i], mv[i], vv[i], s);
            top_m = std::max(top_m, magnitude_bits(mv[i]));
            top_v = std::max(top_v, magnitude_bits(vv[i]));
        }
        m_exp[b] = (uint8_t)shared_exponent(top_m, SPAN_M);
        v_exp[b] = (uint8_t)shared_exponent(top_v, SPAN_V);
        for (int i = 0; i < BLOCK; ++i) {
            const uint32_t u = rounding((uint32_t)((first + b) * BLOCK + i), s.salt);
            m[base + i] = encode_m(mv[i], m_exp[b], u & 0xFFFFu);
            v[base + i] = encode_v(vv[i], v_exp[b], u >> 16);
        }
    });
}

inline void cpu_adamw8_values(const uint8_t* code, const uint8_t* exponent, float* out, int64_t blocks,
                              bool first_moment) {
    for (int64_t i = 0; i < blocks * BLOCK; ++i)
        out[i] = first_moment ? decode_m(code[i], exponent[i / BLOCK]) : decode_v(code[i], exponent[i / BLOCK]);
}

}  // namespace repro_adamw
