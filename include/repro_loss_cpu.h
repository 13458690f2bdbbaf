#pragma once
// repro_loss_cpu.h -- the reproducible softmax cross entropy of a vocabulary projection with its
// gradients on the host CPU (header-only C++17; no GPU needed), bit-identical to
// rg_linear_cross_entropy (include/repro_loss.h), whose arguments cpu_linear_cross_entropy takes.
// Sizes and pointers are not checked (the binding does).
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <vector>

#include "repro_gemm_cpu.h"
#include "repro_loss.h"
#include "repro_loss_math.h"

namespace repro_loss {

namespace cpu_detail {

// Balanced tree over n values, first level v[i] + v[i + n / 2].
template <class T>
T halves(T* v, int n) {
    for (int h = n / 2; h > 0; h /= 2)
        for (int i = 0; i < h; ++i) v[i] = v[i] + v[i + h];
    return v[0];
}

inline void largest_and_sum(const float* z, int V, float& m, float& s) {
    const int parts = (V + PART - 1) / PART;
    std::vector<float> a(parts), b(parts);
    for (int p = 0; p < parts; ++p) {
        const float* q = z + (size_t)p * PART;
        const int n = std::min(PART, V - p * PART);
        a[p] = q[0];
        for (int i = 1; i < n; ++i) a[p] = std::fmax(a[p], q[i]);
        float chunk[PART / 4];
        for (int c = 0; c < PART / 4; ++c) {
            float e[4];
            for (int i = 0; i < 4; ++i) e[i] = 4 * c + i < n ? exp_nonpositive(q[4 * c + i] - a[p]) : 0.0f;
            chunk[c] = (e[0] + e[1]) + (e[2] + e[3]);
        }
        b[p] = a[p] == -INFINITY ? 0.0f : halves(chunk, PART / 4);
    }
    m = a[0];
    for (int p = 1; p < parts; ++p) m = std::fmax(m, a[p]);
    float strand[64] = {};
    for (int p = 0; p < parts; ++p) strand[p % 64] = strand[p % 64] + b[p] * exp_nonpositive(a[p] - m);
    s = halves(strand, 64);
}

inline bool all_finite(const float* v, size_t n) {
    for (size_t i = 0; i < n; ++i)
        if (!finite_bits(v[i])) return false;
    return true;
}

}  // namespace cpu_detail

inline void cpu_linear_cross_entropy(const rg_loss_config& c, const float* x, const float* w, const int64_t* target,
                                     const float* factors, float* loss, float* dx, float* dw) {
    const int64_t N = c.N;
    const int D = c.D, V = c.V;
    int64_t count = 0;
    for (int64_t n = 0; n < N; ++n) count += target[n] != c.ignore_index;
    const float weight = c.reduction == RG_LOSS_MEAN ? 1.0f / (float)count : 1.0f;
    std::vector<char> finite(V);  // the weight's words
    repro_gemm::cpu_for(V, [&](int v) { finite[v] = cpu_detail::all_finite(w + (size_t)v * D, D); });
    const bool finite_weight = std::find(finite.begin(), finite.end(), 0) == finite.end();
    std::vector<Token> tokens(N);
    std::vector<float> z, part, counted;
    const int64_t group = group_tokens(V);
    if (dw) std::fill(dw, dw + (size_t)V * D, 0.0f);
    for (int64_t first = 0; first < N; first += group) {
        const int rows = (int)std::min<int64_t>(group, N - first);
        const float* xg = x + first * D;
        z.resize((size_t)rows * V);
        repro_gemm::cpu_gemm(xg, w, z.data(), rows, V, D, false, true, c.slices);
        repro_gemm::cpu_for_fused(rows, [&](int r) {
            float* q = z.data() + (size_t)r * V;
            Token& t = tokens[first + r];
            const int64_t word = target[first + r];
            const float g = factors ? factors[first + r] : weight;
            t = ignored_token();
            if (word >= 0 && word < V && word != c.ignore_index) {
                if (finite_weight && cpu_detail::all_finite(xg + (size_t)r * D, D)) {
                    float m, s;
                    cpu_detail::largest_and_sum(q, V, m, s);
                    t = finish_token(m, s, q[word], g);
                } else {
                    t = broken_token();
                }
                for (int v = 0; v < V; ++v) q[v] = dz_of(q[v], t.top, t.factor);
                q[word] = 0.0f;
            } else {
                if (word != c.ignore_index) t.loss = NAN;
                std::fill(q, q + V, 0.0f);
            }
        });
        if (dx) {
            float* out = dx + first * D;
            repro_gemm::cpu_gemm(z.data(), w, out, rows, D, V, false, false, c.slices);
            repro_gemm::cpu_for(rows, [&](int r) {
                const int64_t word = target[first + r];
                if (word < 0 || word >= V || word == c.ignore_index) return;
                for (int i = 0; i < D; ++i)
                    out[(size_t)r * D + i] += tokens[first + r].target * w[(size_t)word * D + i];
            });
        }
        if (dw) {
            float* out = first == 0 ? dw : (part.resize((size_t)V * D), part.data());
            counted.assign(xg, xg + (size_t)rows * D);
            for (int r = 0; r < rows; ++r)
                if (tokens[first + r].factor == 0.0f) std::fill_n(counted.begin() + (size_t)r * D, D, 0.0f);
            repro_gemm::cpu_gemm(z.data(), counted.data(), out, V, D, rows, true, false, c.slices);
            if (first > 0)
                for (size_t i = 0; i < (size_t)V * D; ++i) dw[i] = dw[i] + part[i];
        }
    }
    if (dw) {  // the target words' rows: their tokens in order, every 16th to one of 16 sums from +0
        std::vector<std::vector<int64_t>> of(V);
        for (int64_t n = 0; n < N; ++n)
            if (target[n] >= 0 && target[n] < V && target[n] != c.ignore_index) of[target[n]].push_back(n);
        repro_gemm::cpu_for(V, [&](int v) {
            if (of[v].empty()) return;
            for (int i = 0; i < D; ++i) {
                float sum[16] = {};
                for (size_t k = 0; k < of[v].size(); ++k)
                    sum[k % 16] = sum[k % 16] + tokens[of[v][k]].target * x[of[v][k] * D + i];
                dw[(size_t)v * D + i] = dw[(size_t)v * D + i] + cpu_detail::halves(sum, 16);
            }
        });
    }
    if (!loss) return;
    std::vector<float> rows(N);
    for (int64_t n = 0; n < N; ++n) rows[n] = tokens[n].loss;
    if (c.reduction == RG_LOSS_NONE) {
        std::copy(rows.begin(), rows.end(), loss);
        return;
    }
    std::vector<double> sum(STRANDS, 0.0);
    for (int64_t n = 0; n < N; ++n) sum[n % STRANDS] = sum[n % STRANDS] + (double)rows[n];
    const double all = cpu_detail::halves(sum.data(), STRANDS);
    loss[0] = (float)(c.reduction == RG_LOSS_MEAN ? all / (double)count : all);
}

}  // namespace repro_loss
