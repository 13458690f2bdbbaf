#pragma once
// repro_norm_cpu.h -- the reproducible residual addition with the norms before and after a block on the
// host CPU (header-only C++17; no GPU needed), bit-identical to rg_residual_norm_fp32 and
// rg_residual_norm_grad_fp32 (include/repro_norm.h), whose arguments these take; `bad`, when not null, is set where
// those lower their flag. Arguments are not checked (the binding does).
#include <atomic>
#include <cmath>
#include <cstdint>
#include <vector>

#include "repro_gemm_cpu.h"
#include "repro_norm.h"
#include "repro_norm_math.h"

namespace repro_norm {

namespace cpu_detail {

// The sum over a row of the D values value(i).
template <class F>
float row_sum(int D, F value) {
    const int S = strands_of(D);
    float s[1024] = {};
    for (int c = 0; 4 * c < D; ++c) {
        float v[4];
        for (int i = 0; i < 4; ++i) v[i] = 4 * c + i < D ? value(4 * c + i) : 0.0f;
        const float q = (v[0] + v[1]) + (v[2] + v[3]);
        s[c % S] = c < S ? q : s[c % S] + q;
    }
    for (int step = 64; step < S; step *= 2)  // neighbours s, s + 64; then s, s + 128; ...
        for (int a = 0; a < S; a += 2 * step)
            for (int l = 0; l < 64; ++l) s[a + l] = s[a + l] + s[a + step + l];
    for (int half = 32; half > 0; half /= 2)
        for (int l = 0; l < half; ++l) s[l] = s[l] + s[l + half];
    return s[0];
}

inline RowStats row_stats(const float* v, int D, float eps, bool layer) {
    RowStats st;
    st.mean = layer ? mean_of(row_sum(D, [&](int i) { return v[i]; }), D) : 0.0f;
    st.rstd = rstd_of(row_sum(D, [&](int i) {
        const float c = centred(v[i], st.mean, layer);
        return c * c;
    }), D, eps);
    return st;
}

inline float tree16(const float* v) {
    float t[16];
    for (int i = 0; i < 16; ++i) t[i] = v[i];
    for (int n = 8; n > 0; n /= 2)
        for (int i = 0; i < n; ++i) t[i] = t[2 * i] + t[2 * i + 1];
    return t[0];
}

// Column i's total of P partials, p-th at part[p * D + i].
inline float total(const float* part, long long P, int D, int i) {
    float phase[16] = {};
    for (long long p = 0; p < P; ++p) phase[p % 16] = phase[p % 16] + part[p * D + i];
    return tree16(phase);
}

}  // namespace cpu_detail

inline void cpu_residual_norm(const rg_norm_config& c, const float* x, const float* f, const float* gate,
                              const float* post_weight, const float* post_bias, const float* weight,
                              const float* bias, float* r, float* y, float* stats, bool* bad = nullptr) {
    std::atomic<bool> found{false};
    const int D = c.D;
    const bool layer = !c.rms;
    const long long group = c.gate_rows > 0 ? c.N / c.gate_rows : 1;
    repro_gemm::cpu_for((int)c.N, [&](int n) {
        const size_t at = (size_t)n * D;
        const float* v = x + at;
        RowStats sf{0.0f, 0.0f};
        if (f) {
            if (c.post) sf = cpu_detail::row_stats(f + at, D, c.eps, layer);
            const float* g = gate ? gate + (size_t)(n / group) * D : nullptr;
            for (int i = 0; i < D; ++i) {
                float u = f[at + i];
                if (c.post)
                    u = affine(centred(u, sf.mean, layer) * sf.rstd, post_weight, post_weight ? post_weight[i] : 0.0f,
                               post_bias, post_bias ? post_bias[i] : 0.0f);
                if (g) u = u * g[i];
                r[at + i] = x[at + i] + u * c.scale;
            }
            v = r + at;
        }
        const RowStats s = cpu_detail::row_stats(v, D, c.eps, layer);
        for (int i = 0; i < D; ++i)
            y[at + i] = affine(centred(v[i], s.mean, layer) * s.rstd, weight, weight ? weight[i] : 0.0f, bias,
                               bias ? bias[i] : 0.0f);
        if (!(s.rstd > 0.0f && (!c.post || sf.rstd > 0.0f))) found.store(true, std::memory_order_relaxed);
        if (stats) {
            stats[4 * (size_t)n] = s.mean;
            stats[4 * (size_t)n + 1] = s.rstd;
            stats[4 * (size_t)n + 2] = sf.mean;
            stats[4 * (size_t)n + 3] = sf.rstd;
        }
    });
    if (bad && found) *bad = true;
}

inline void cpu_residual_norm_grad(const rg_norm_config& c, const float* dr, const float* dy, const float* r,
                                   const float* f, const float* gate, const float* post_weight,
                                   const float* post_bias, const float* weight, const float* stats, float* dx,
                                   float* df, float* dgate, float* dpost_weight, float* dpost_bias,
                                   float* dweight, float* dbias, bool* bad = nullptr) {
    std::atomic<bool> found{false};
    const int D = c.D;
    const bool layer = !c.rms;
    const Partition pt = partition(c.N, D, c.gate_rows);
    const long long P = pt.sections * pt.partials;
    enum { W, B, PW, PB, GATE, SUMS };
    std::vector<float> part((size_t)SUMS * P * D, 0.0f);
    repro_gemm::cpu_for((int)P, [&](int p) {
        const long long section = p / pt.partials, p_in = p % pt.partials;
        std::vector<float> strand((size_t)pt.join * SUMS * D, 0.0f), a(D), hat(D), u(D), fhat(D);
        for (int j = 0; j < pt.join; ++j) {
            float* s = strand.data() + (size_t)j * SUMS * D;
            const long long first = (p_in * pt.join + j) * pt.rows;
            const long long end = std::min(first + pt.rows, pt.section_rows);
            for (long long k = first; k < end; ++k) {
                const long long n = section * pt.section_rows + k;
                const size_t at = (size_t)n * D;
                const float *st = stats + 4 * n, *g = gate ? gate + (size_t)(n / pt.group_rows) * D : nullptr;
                for (int i = 0; i < D; ++i) hat[i] = centred(r[at + i], st[0], layer) * st[1];
                float c1 = 0.0f, c2 = 0.0f;
                if (dy) {
                    for (int i = 0; i < D; ++i) {
                        a[i] = weight ? dy[at + i] * weight[i] : dy[at + i];
                        s[W * D + i] = s[W * D + i] + dy[at + i] * hat[i];
                        s[B * D + i] = s[B * D + i] + dy[at + i];
                    }
                    if (layer) c1 = mean_of(cpu_detail::row_sum(D, [&](int i) { return a[i]; }), D);
                    c2 = mean_of(cpu_detail::row_sum(D, [&](int i) { return a[i] * hat[i]; }), D);
                }
                for (int i = 0; i < D; ++i) {
                    float d = dr ? dr[at + i] : 0.0f;
                    if (dy) {
                        const float b = backward(a[i], hat[i], st[1], c1, c2, layer);
                        d = dr ? d + b : b;
                    }
                    if (dx) dx[at + i] = d;
                    if (!std::isfinite(d)) found.store(true, std::memory_order_relaxed);
                    a[i] = d * c.scale;
                }
                if (!f) continue;
                for (int i = 0; i < D; ++i) {
                    fhat[i] = c.post ? centred(f[at + i], st[2], layer) * st[3] : 0.0f;
                    u[i] = c.post ? affine(fhat[i], post_weight, post_weight ? post_weight[i] : 0.0f, post_bias,
                                           post_bias ? post_bias[i] : 0.0f)
                                  : f[at + i];
                    if (g) {
                        s[GATE * D + i] = s[GATE * D + i] + a[i] * u[i];
                        a[i] = a[i] * g[i];
                    }
                }
                if (g && pt.gate_inside && (k + 1) % pt.group_rows == 0) {
                    for (int i = 0; i < D; ++i) {
                        if (dgate) dgate[(size_t)(n / pt.group_rows) * D + i] = s[GATE * D + i];
                        s[GATE * D + i] = 0.0f;
                    }
                }
                if (c.post) {
                    for (int i = 0; i < D; ++i) {
                        s[PW * D + i] = s[PW * D + i] + a[i] * fhat[i];
                        s[PB * D + i] = s[PB * D + i] + a[i];
                        if (post_weight) a[i] = a[i] * post_weight[i];
                    }
                    c1 = layer ? mean_of(cpu_detail::row_sum(D, [&](int i) { return a[i]; }), D) : 0.0f;
                    c2 = mean_of(cpu_detail::row_sum(D, [&](int i) { return a[i] * fhat[i]; }), D);
                    for (int i = 0; i < D; ++i) a[i] = backward(a[i], fhat[i], st[3], c1, c2, layer);
                }
                if (df)
                    for (int i = 0; i < D; ++i) df[at + i] = a[i];
            }
        }
        for (int q = 0; q < SUMS; ++q) {
            for (int i = 0; i < D; ++i) {
                float v[4];
                for (int j = 0; j < pt.join; ++j) v[j] = strand[((size_t)j * SUMS + q) * D + i];
                part[((size_t)q * P + p) * D + i] = pt.join == 4 ? (v[0] + v[1]) + (v[2] + v[3]) : v[0];
            }
        }
    });
    if (bad && found) *bad = true;
    float* out[] = {dweight, dbias, dpost_weight, dpost_bias};
    for (int q = W; q <= PB; ++q)
        if (out[q])
            for (int i = 0; i < D; ++i) out[q][i] = cpu_detail::total(part.data() + (size_t)q * P * D, P, D, i);
    if (dgate && !pt.gate_inside)
        for (long long s = 0; s < pt.sections; ++s)
            for (int i = 0; i < D; ++i)
                dgate[s * D + i] =
                    cpu_detail::total(part.data() + ((size_t)GATE * P + s * pt.partials) * D, pt.partials, D, i);
}

}  // namespace repro_norm
