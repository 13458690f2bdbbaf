#pragma once
// repro_attention_cpu.h -- the reproducible attention with its gradients and the bias of relative positions on the
// host CPU (header-only C++17; no GPU needed), bit-identical to include/repro_attention.h's entries,
// whose arguments these take (the mask packed to words of 64 keys). Arguments are not checked (the binding does).
#include <cmath>
#include <cstdint>
#include <vector>

#include "repro_attention.h"
#include "repro_attention_math.h"
#include "repro_dropout_math.h"
#include "repro_gemm_cpu.h"

namespace repro_attention {

namespace cpu_detail {

// run(n) for every n in [0, count), spread over the workers.
template <class F>
void spread(long long count, F run) {
    const long long parts = count < (1 << 20) ? count : 1 << 20;
    repro_gemm::cpu_for_fused((int)parts, [&](int part) {
        for (long long n = part; n < count; n += parts) run(n);
    });
}

struct Call {
    const rg_attention_config& c;
    const float *q, *k, *v;
    const long long* key_lengths;
    const unsigned long long* mask;
    const float* bias;
    float factor = score_factor(c.scale);
    float keep_factor = repro_dropout::factor_of(c.dropout);
    uint32_t threshold = repro_dropout::threshold_of(c.dropout);
    long long words = (c.Tk + 63) / 64;
    long long start = c.query_start > c.Tk ? c.Tk : c.query_start < -c.Tq ? -c.Tq : c.query_start;  // past the ends nothing changes

    const float* row(const float* p, const long long* s, long long b, long long n, long long h) const {
        return p + b * s[0] + n * s[1] + h * s[2];
    }
    const float* query(long long b, long long h, long long i) const { return row(q, c.q_stride, b, i, h); }
    const float* key(long long b, long long h, long long j) const { return row(k, c.k_stride, b, j, h / (c.H / c.KVH)); }
    const float* value(long long b, long long h, long long j) const { return row(v, c.v_stride, b, j, h / (c.H / c.KVH)); }
    // The keys from which on query i sees none, the mask aside.
    long long end(long long b, long long i) const {
        long long n = c.Tk;
        if (key_lengths && key_lengths[b] < n) n = key_lengths[b];
        if (c.causal && i + start + 1 < n) n = i + start + 1;
        return n < 0 ? 0 : n;
    }
    bool seen(long long b, long long h, long long i, long long j) const {
        if (j >= end(b, i)) return false;
        if (!mask) return true;
        const unsigned long long* m = mask + b * c.mask_stride[0] + h * c.mask_stride[1] + i * c.mask_stride[2];
        return (m[j >> 6] >> (j & 63) & 1) != 0;
    }
    static float dot(const float* a, const float* b, int D) {
        float s = 0.0f;
        for (int d = 0; d < D; ++d) s = __builtin_fmaf(a[d], b[d], s);
        return s;
    }
    // t, and its difference to a maximum.
    struct Score {
        float s, t;
        bool biased;
        float factor;
        float less(float base) const { return repro_attention::less(s, t, factor, base, biased); }
    };
    Score score(long long b, long long h, long long i, long long j) const {
        const float s = dot(query(b, h, i), key(b, h, j), c.D);
        if (!bias) return Score{s, s * factor, false, factor};
        return Score{s, __builtin_fmaf(s, factor, bias_term(bias[h * (c.Tq + c.Tk - 1) + j - i + c.Tq - 1])), true, factor};
    }
    bool kept(long long b, long long h, long long i, long long j) const {
        if (threshold == 0) return true;
        const auto w = repro_dropout::pair_words((uint32_t)(j / 4), (uint32_t)i, (uint32_t)(b * c.H + h), c.seed);
        return w.w[j % 4] >= threshold;
    }
};

inline void forward_row(const Call& z, long long b, long long h, long long i, float* y, float* stats) {
    const int D = z.c.D;
    float top = NONE, total = 0.0f, out[MAX_D] = {};
    const long long end = z.end(b, i);
    for (long long first = 0; first < end; first += CHUNK) {
        float m = NONE, l[2] = {0.0f, 0.0f}, o[MAX_D] = {};
        for (long long j0 = first; j0 < first + CHUNK && j0 < end; j0 += TILE) {
            Call::Score t[TILE];
            float next = m;
            bool seen[TILE];
            for (int n = 0; n < TILE; ++n) {
                seen[n] = j0 + n < end && z.seen(b, h, i, j0 + n);
                if (!seen[n]) continue;
                t[n] = z.score(b, h, i, j0 + n);
                next = larger(next, t[n].t);
            }
            const float a = rescale(m, base_of(next));
            m = next;
            for (float& x : l) x = x * a;
            for (int d = 0; d < D; ++d) o[d] = o[d] * a;
            for (int n = 0; n < TILE; ++n) {
                if (!seen[n]) continue;
                const float p = e2(t[n].less(base_of(m)));
                l[n & 1] = l[n & 1] + p;
                const float u = z.kept(b, h, i, j0 + n) ? p : 0.0f;
                const float* v = z.value(b, h, j0 + n);
                for (int d = 0; d < D; ++d) o[d] = __builtin_fmaf(u, v[d], o[d]);
            }
        }
        const float both = larger(top, m), a = rescale(top, base_of(both)), e = rescale(m, base_of(both));
        top = both;
        total = __builtin_fmaf(l[0] + l[1], e, total * a);
        for (int d = 0; d < D; ++d) out[d] = __builtin_fmaf(o[d], e, out[d] * a);
    }
    const float inverse = reciprocal(total);
    const float f = z.threshold == 0 ? inverse : inverse * z.keep_factor;
    for (int d = 0; d < D; ++d) y[d] = out[d] * f + 0.0f;  // (no -0)
    if (stats) {
        stats[0] = base_of(top);
        stats[1] = inverse;
    }
}

}  // namespace cpu_detail

inline void cpu_pack_mask(const unsigned char* mask, long long items, long long heads, long long queries, long long Tk,
                          const long long stride[3], long long key_stride, unsigned long long* words) {
    const long long W = (Tk + 63) / 64;
    cpu_detail::spread(items * heads * queries, [&](long long n) {
        const long long i = n % queries, h = n / queries % heads, b = n / queries / heads;
        const unsigned char* m = mask + b * stride[0] + h * stride[1] + i * stride[2];
        for (long long w = 0; w < W; ++w) {
            unsigned long long bits = 0;
            for (int k = 0; k < 64 && 64 * w + k < Tk; ++k) bits |= (unsigned long long)(m[(64 * w + k) * key_stride] != 0) << k;
            words[n * W + w] = bits;
        }
    });
}

inline void cpu_attention(const rg_attention_config& c, const float* q, const float* k, const float* v,
                          const long long* key_lengths, const unsigned long long* mask, const float* bias, float* y,
                          float* stats) {
    const cpu_detail::Call z{c, q, k, v, key_lengths, mask, bias};
    cpu_detail::spread(c.B * c.H * c.Tq, [&](long long n) {
        const long long i = n % c.Tq, h = n / c.Tq % c.H, b = n / c.Tq / c.H;
        cpu_detail::forward_row(z, b, h, i, y + ((b * c.Tq + i) * c.H + h) * c.D, stats ? stats + 2 * n : nullptr);
    });
}

inline void cpu_attention_grad(const rg_attention_config& c, const float* dy, const float* q, const float* k, const float* v,
                               const long long* key_lengths, const unsigned long long* mask, const float* bias, const float* y,
                               const float* stats, float* dq, float* dk, float* dv, float* dbias) {
    const cpu_detail::Call z{c, q, k, v, key_lengths, mask, bias};
    const int D = c.D, group = c.H / c.KVH;
    const float scale = (float)c.scale;
    const auto place = [&](long long b, long long i, long long h) { return ((b * c.Tq + i) * c.H + h) * (long long)D; };
    std::vector<float> delta((size_t)(c.B * c.H * c.Tq));
    cpu_detail::spread(c.B * c.H * c.Tq, [&](long long n) {
        const long long i = n % c.Tq, h = n / c.Tq % c.H, b = n / c.Tq / c.H;
        const float *a = dy + place(b, i, h), *o = y + place(b, i, h);
        float s[64];
        for (int l = 0; l < 64; ++l) {
            s[l] = l < D ? a[l] * o[l] : 0.0f;
            s[l] = l + 64 < D ? __builtin_fmaf(a[l + 64], o[l + 64], s[l]) : s[l];
        }
        for (int half = 32; half > 0; half /= 2)
            for (int l = 0; l < half; ++l) s[l] = s[l] + s[l + half];
        delta[n] = s[0];
    });
    struct Pair {
        float u, ds;
    };
    const auto pair = [&](long long b, long long h, long long i, long long j) {
        const long long n = (b * c.H + h) * c.Tq + i;
        const float p = e2(z.score(b, h, i, j).less(stats[2 * n])) * stats[2 * n + 1];
        float u = p, dp = cpu_detail::Call::dot(dy + place(b, i, h), z.value(b, h, j), D);
        if (z.threshold != 0) {
            const bool kept = z.kept(b, h, i, j);
            u = kept ? p * z.keep_factor : 0.0f;
            dp = kept ? dp * z.keep_factor : 0.0f;
        }
        return Pair{u, ds_of(p, dp, delta[n])};
    };
    cpu_detail::spread(c.B * c.KVH * c.Tk, [&](long long n) {
        const long long j = n % c.Tk, g = n / c.Tk % c.KVH, b = n / c.Tk / c.KVH;
        float sv[MAX_D] = {}, sk[MAX_D] = {};
        for (long long h = g * group; h < (g + 1) * group; ++h) {
            float hv[MAX_D] = {}, hk[MAX_D] = {};
            for (long long first = 0; first < c.Tq; first += QUERY_CHUNK) {
                float pv[MAX_D] = {}, pk[MAX_D] = {};
                for (long long i = first; i < first + QUERY_CHUNK && i < c.Tq; ++i) {
                    if (!z.seen(b, h, i, j)) continue;
                    const Pair w = pair(b, h, i, j);
                    const float *a = dy + place(b, i, h), *x = z.query(b, h, i);
                    for (int d = 0; d < D; ++d) pv[d] = __builtin_fmaf(w.u, a[d], pv[d]);
                    for (int d = 0; d < D; ++d) pk[d] = __builtin_fmaf(w.ds, x[d], pk[d]);
                }
                for (int d = 0; d < D; ++d) hv[d] = hv[d] + pv[d];
                for (int d = 0; d < D; ++d) hk[d] = hk[d] + pk[d];
            }
            for (int d = 0; d < D; ++d) sv[d] = sv[d] + hv[d];
            for (int d = 0; d < D; ++d) sk[d] = sk[d] + hk[d];
        }
        const long long at = ((b * c.Tk + j) * c.KVH + g) * D;
        for (int d = 0; d < D; ++d) {
            dv[at + d] = sv[d] + 0.0f;
            dk[at + d] = sk[d] * scale + 0.0f;
        }
    });
    cpu_detail::spread(c.B * c.H * c.Tq, [&](long long n) {
        const long long i = n % c.Tq, h = n / c.Tq % c.H, b = n / c.Tq / c.H;
        const long long end = z.end(b, i);
        float s[MAX_D] = {};
        for (long long first = 0; first < end; first += KEY_BLOCK) {
            float part[MAX_D] = {};
            for (long long j = first; j < first + KEY_BLOCK && j < end; ++j) {
                if (!z.seen(b, h, i, j)) continue;
                const float ds = pair(b, h, i, j).ds;
                const float* x = z.key(b, h, j);
                for (int d = 0; d < D; ++d) part[d] = __builtin_fmaf(ds, x[d], part[d]);
            }
            for (int d = 0; d < D; ++d) s[d] = s[d] + part[d];
        }
        for (int d = 0; d < D; ++d) dq[place(b, i, h) + d] = s[d] * scale + 0.0f;
    });
    if (!dbias) return;
    const long long columns = c.Tq + c.Tk - 1;
    cpu_detail::spread(c.H * columns, [&](long long n) {
        const long long h = n / columns, away = n % columns - (c.Tq - 1);
        float s = 0.0f;
        for (long long block = 0; block < c.Tk; block += KEY_BLOCK)
            for (long long b = 0; b < c.B; ++b)
                for (long long first = 0; first < c.Tq; first += QUERY_CHUNK) {
                    const long long high = std::min(block + KEY_BLOCK, c.Tk);
                    long long i = std::max(first, block - away), last = std::min({first + QUERY_CHUNK, c.Tq, high - away});
                    if (i >= last) continue;
                    float part = 0.0f;
                    for (; i < last; ++i)
                        if (z.seen(b, h, i, i + away)) part = part + pair(b, h, i, i + away).ds;
                    s = s + part;
                }
        dbias[n] = s + 0.0f;
    });
}

inline float cpu_tree(float* s, int n) {
    for (int half = n / 2; half > 0; half /= 2)
        for (int l = 0; l < half; ++l) s[l] = s[l] + s[l + half];
    return s[0];
}

inline void cpu_relative_bias(const rg_relative_bias_config& c, const float* table, float* out) {
    const long long columns = c.Tq + c.Tk - 1, rows = c.dense ? c.Tq : 1, width = c.dense ? c.Tk : columns;
    cpu_detail::spread(c.H * rows, [&](long long n) {
        const long long h = n / rows, i = n % rows;
        for (long long x = 0; x < width; ++x) {
            const long long away = c.dense ? x - i : x - (c.Tq - 1);
            out[n * width + x] = table[bucket_of(away - c.query_start, c.borders, c.count, c.both) * (long long)c.H + h];
        }
    });
}

inline void cpu_relative_bias_grad(const rg_relative_bias_config& c, const float* dout, float* dtable) {
    const long long columns = c.Tq + c.Tk - 1;
    const int buckets = (c.count + 1) * (c.both ? 2 : 1);
    std::vector<float> by_distance;
    if (c.dense) {
        by_distance.resize((size_t)(c.H * columns));
        cpu_detail::spread(c.H * columns, [&](long long n) {
            const long long h = n / columns, away = n % columns - (c.Tq - 1);
            float s = 0.0f;
            for (long long first = 0; first < c.Tq; first += RUN) {
                float part = 0.0f;
                for (long long i = std::max(first, -away); i < std::min({first + RUN, c.Tq, c.Tk - away}); ++i)
                    part = part + dout[(h * c.Tq + i) * c.Tk + i + away];
                s = s + part;
            }
            by_distance[n] = s;
        });
        dout = by_distance.data();
    }
    cpu_detail::spread((long long)buckets * c.H, [&](long long n) {
        const long long bucket = n / c.H, h = n % c.H;
        float s[STRANDS] = {};
        for (long long x = 0; x < columns; ++x)
            if (bucket_of(x - (c.Tq - 1) - c.query_start, c.borders, c.count, c.both) == bucket)
                s[x % STRANDS] = s[x % STRANDS] + dout[h * columns + x];
        dtable[n] = cpu_tree(s, STRANDS) + 0.0f;
    });
}

}  // namespace repro_attention
