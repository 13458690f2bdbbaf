// Host build of the attention's exponential (include/repro_attention_math.h), for its error bound.
#include <cmath>
#include <cstdint>

#include "repro_attention_math.h"
#include "repro_gemm_cpu.h"

extern "C" {

float ha_e2(float x) { return repro_attention::e2(x); }

// The largest error over every step-th float between the bit patterns lo and hi: in units of the result's last place (results from 2^-126
// up), relative to it, and of results below 2^-126 in units of 2^-149.
void ha_e2_errors(uint32_t lo, uint32_t hi, uint32_t step, double* units, double* relative, double* below) {
    *units = *relative = *below = 0.0;
    for (uint64_t b = lo; b < hi; b += step) {
        const float x = repro_gemm::bits_to_float((uint32_t)b);
        const double want = std::exp2((double)x), off = std::fabs((double)repro_attention::e2(x) - want);
        if (want < 0x1p-126) {
            *below = std::fmax(*below, off * 0x1p149);
            continue;
        }
        int e;
        std::frexp(want, &e);
        *units = std::fmax(*units, off / std::ldexp(1.0, e - 24));
        *relative = std::fmax(*relative, off / want);
    }
}

// out[i]: a chain of n fused multiply-adds and exponentials of a[i], by cpu_for_fused or by cpu_for.
void ha_chains(const float* a, float* out, int count, int n, int fused) {
    const auto run = [&](int i) {
        float s = a[i];
        for (int k = 0; k < n; ++k) s = __builtin_fmaf(s, a[i], repro_attention::e2(-s * s));
        out[i] = s;
    };
    if (fused) repro_gemm::cpu_for_fused(count, run);
    else repro_gemm::cpu_for(count, run);
}

}  // extern "C"
