#pragma once
// repro_dropout_cpu.h -- the reproducible dropout on the host CPU (header-only C++17; no GPU needed), bit-identical
// to rg_dropout_fp32 (include/repro_dropout.h).
#include "repro_dropout_math.h"
#include "repro_gemm_cpu.h"

namespace repro_dropout {

inline void cpu_dropout(const float* x, float* y, size_t n, double p, uint64_t seed) {
    const uint32_t threshold = threshold_of(p);
    const float factor = factor_of(p);
    const size_t groups = (n + 3) / 4, run = 4096;
    repro_gemm::cpu_for((int)((groups + run - 1) / run), [&](int part) {
        const size_t end = std::min(groups, ((size_t)part + 1) * run);
        for (size_t g = (size_t)part * run; g < end; ++g) {
            const Words r = value_words(g, seed);
            for (int i = 0; i < 4 && 4 * g + i < n; ++i) y[4 * g + i] = r.w[i] >= threshold ? x[4 * g + i] * factor : 0.0f;
        }
    });
}

}  // namespace repro_dropout
