// The residual addition with the norms before and after a block, and its gradients, each in one read of
// its rows.
//
// WAVES wavefronts hold a row in registers, 4 NK values a thread (chunk c of 4 consecutive values at
// thread c mod 64 WAVES), so a row is read once and its mean, its centred squares and its outputs are
// taken from there. A row of at most 1024 values is one wavefront's, whose sums need no barrier; wider
// ones take 8 or 16, which hold the next row while they work on one.
//
// HBM bounds both passes: 16 bytes a value forward (x, f, r, y) and 16 to 24 backward (dr, dy, r, dx, and f and df).
// 8192 rows of 768: 17.3 us forward (101 MB, partly in the caches: 5.8 TB/s) and 23.2 backward. 4096 rows of
// 4096 with both norms and a gate: 56 and 91 us, 4.8 and 4.4 TB/s, where a copy of 1 GiB reaches 5.1 (with loads
// and stores past the caches 53 and 88, but 19.6 and 26.8 for the 8192 rows of 768, which find each other's rows
// there). Sums over rows (the weights' gradients) stay in registers over a block's rows and meet in norm_totals, 4 to 7 us.
#include "rg_internal.h"
#include "repro_norm.h"
#include "repro_norm_math.h"

#include <cmath>
#include <cstdint>

namespace rg {
namespace {

using repro_norm::affine;
using repro_norm::backward;
using repro_norm::centred;
using repro_norm::mean_of;
using repro_norm::Partition;

// 16 bytes at a multiple of 4: rows whose length is no multiple of 4 start anywhere.
struct __attribute__((packed, aligned(4))) Four {
    float v[4];
};

template <int T, int NK>
struct Chunks {
    float v[NK][4];

    __device__ __forceinline__ void load(const float* __restrict__ p, int D, int t) {
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const int at = 4 * (t + T * k);
            if (at + 4 <= D) {
                const Four q = *reinterpret_cast<const Four*>(p + at);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[k][i] = q.v[i];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[k][i] = at + i < D ? p[at + i] : 0.0f;
            }
        }
    }
    __device__ __forceinline__ void store(float* __restrict__ p, int D, int t) const {
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const int at = 4 * (t + T * k);
            if (at + 4 <= D) {
                Four q;
#pragma unroll
                for (int i = 0; i < 4; ++i) q.v[i] = v[k][i];
                *reinterpret_cast<Four*>(p + at) = q;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at + i < D) p[at + i] = v[k][i];
            }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[k][i] = 0.0f;
    }
};

template <int CTRL>
__device__ __forceinline__ float rotated(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}

// v + its partner 32 lanes away, then 16, 8, ..., 1: the sum over the wavefront, in every lane. The
// half-wave and row swaps give both partners of a pair to both; within a row of 16 a rotation by n finds
// a partner's sum, as the sums repeat every 2 n lanes by then.
__device__ __forceinline__ float wave_sum(float v) {
    auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    v = v + rotated<0x128>(v);
    v = v + rotated<0x124>(v);
    v = v + rotated<0x122>(v);
    return v + rotated<0x121>(v);
}

// Sums over a row, in the order of repro_norm_math.h. One wavefront needs no exchange. With as many threads as
// strands a thread holds a strand; with twice as many, its chunks are added after the exchange. `turn`
// alternates the exchange's halves, so one barrier a sum is enough.
template <int WAVES, int NK>
struct RowSum {
    static constexpr int T = 64 * WAVES, CHUNKS = T * NK;
    static constexpr int STRANDS = CHUNKS <= 1024 ? 256 : 1024;  // a row of at most 4096 values: 256
    static constexpr bool JOINED = T <= STRANDS;                 // a thread adds up its strand itself
    static constexpr int HELD = JOINED ? T : CHUNKS;             // values exchanged for a sum
    static constexpr int LDS = WAVES == 1 ? 1 : 4 * HELD;
    float* lds;  // LDS floats
    int t, D, turn;

    template <class F>
    __device__ __forceinline__ float chunk(int k, F value) const {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = 4 * (t + T * k) + i < D ? value(k, i) : 0.0f;
        return (v[0] + v[1]) + (v[2] + v[3]);
    }
    template <class F>
    __device__ __forceinline__ void put(float* __restrict__ p, F value) const {
        if constexpr (JOINED) {
            float s = chunk(0, value);
#pragma unroll
            for (int k = 1; k < NK; ++k) {
                const float q = chunk(k, value);
                s = 4 * (t + T * k) < D ? s + q : s;
            }
            p[t] = s;
        } else {
#pragma unroll
            for (int k = 0; k < NK; ++k) p[t + T * k] = chunk(k, value);
        }
    }
    __device__ __forceinline__ float take(const float* __restrict__ p) const {
        constexpr int N = JOINED ? WAVES : STRANDS / 64;
        const int lane = t & 63;
        float v[N];
#pragma unroll
        for (int w = 0; w < N; ++w) {
            v[w] = p[64 * w + lane];
            if constexpr (!JOINED) {
#pragma unroll
                for (int c = STRANDS; c < CHUNKS; c += STRANDS) {
                    const float q = p[c + 64 * w + lane];
                    v[w] = 4 * (c + 64 * w + lane) < D ? v[w] + q : v[w];
                }
            }
        }
#pragma unroll
        for (int n = N / 2; n > 0; n /= 2)
#pragma unroll
            for (int w = 0; w < n; ++w) v[w] = v[2 * w] + v[2 * w + 1];
        return wave_sum(v[0]);
    }
    template <class F>
    __device__ __forceinline__ float one(F value) {
        if constexpr (WAVES == 1) {
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < NK; ++k) s[k] = chunk(k, value);
            return wave_sum((s[0] + s[1]) + (s[2] + s[3]));
        } else {
            float* p = lds + turn * 2 * HELD;
            turn ^= 1;
            put(p, value);
            __syncthreads();
            return take(p);
        }
    }
    template <class F, class G>
    __device__ __forceinline__ void two(F f, G g, float& a, float& b) {
        if constexpr (WAVES == 1) {
            a = one(f);
            b = one(g);
        } else {
            float* p = lds + turn * 2 * HELD;
            turn ^= 1;
            put(p, f);
            put(p + HELD, g);
            __syncthreads();
            a = take(p);
            b = take(p + HELD);
        }
    }
};

struct Sizes {
    long long N;
    int D;
    float eps, scale;
    bool layer;
};

template <int WAVES, int NK>
__device__ __forceinline__ repro_norm::RowStats stats_of(const Chunks<64 * WAVES, NK>& v, RowSum<WAVES, NK>& sum,
                                                         const Sizes& z) {
    repro_norm::RowStats st;
    st.mean = z.layer ? mean_of(sum.one([&](int k, int i) { return v.v[k][i]; }), z.D) : 0.0f;
    const float squares = sum.one([&](int k, int i) {
        const float c = centred(v.v[k][i], st.mean, z.layer);
        return c * c;
    });
    st.rstd = repro_norm::rstd_of(squares, z.D, z.eps);
    return st;
}

__device__ __forceinline__ void report(int* flag, int op_id) { atomicMin(flag, op_id); }

template <int WAVES, int NK, bool POST>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES)
norm_forward(Sizes z, long long group, const float* __restrict__ x, const float* __restrict__ f,
             const float* __restrict__ gate, const float* __restrict__ post_weight,
             const float* __restrict__ post_bias, const float* __restrict__ weight,
             const float* __restrict__ bias, float* __restrict__ r, float* __restrict__ y,
             float* __restrict__ stats, int* flag, int op_id) {
    constexpr int T = 64 * WAVES, ROWS = WAVES == 1 ? 4 : 1;
    __shared__ float lds[RowSum<WAVES, NK>::LDS];
    const int t = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    RowSum<WAVES, NK> sum{lds, t, z.D, 0};
    const int sub = WAVES == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const long long step = (long long)gridDim.x * ROWS;
    constexpr bool AHEAD = WAVES > 1;  // the next row's values are in flight while a row is worked on
    Chunks<T, NK> next_x, next_f;
    const auto fetch = [&](long long n) {
        if (n >= z.N) return;
        next_x.load(x + (size_t)n * z.D, z.D, t);
        if (f != nullptr) next_f.load(f + (size_t)n * z.D, z.D, t);
    };
    long long n = (long long)blockIdx.x * ROWS + sub;
    if (AHEAD) fetch(n);
    for (; n < z.N; n += step) {
        const size_t at = (size_t)n * z.D;
        if (!AHEAD) fetch(n);
        Chunks<T, NK> v = next_x, u = next_f, w;
        if (AHEAD) fetch(n + step);
        repro_norm::RowStats sf{0.0f, 0.0f};
        if (f != nullptr) {
            if constexpr (POST) {
                sf = stats_of<WAVES, NK>(u, sum, z);
                Chunks<T, NK> b;
                if (post_weight != nullptr) w.load(post_weight, z.D, t);
                if (post_bias != nullptr) b.load(post_bias, z.D, t);
#pragma unroll
                for (int k = 0; k < NK; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        u.v[k][i] = affine(centred(u.v[k][i], sf.mean, z.layer) * sf.rstd, post_weight != nullptr,
                                           w.v[k][i], post_bias != nullptr, b.v[k][i]);
            }
            if (gate != nullptr) {
                w.load(gate + (size_t)(n / group) * z.D, z.D, t);
#pragma unroll
                for (int k = 0; k < NK; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) u.v[k][i] = u.v[k][i] * w.v[k][i];
            }
#pragma unroll
            for (int k = 0; k < NK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) v.v[k][i] = v.v[k][i] + u.v[k][i] * z.scale;
            v.store(r + at, z.D, t);
        }
        const repro_norm::RowStats s = stats_of<WAVES, NK>(v, sum, z);
        Chunks<T, NK> b;
        if (weight != nullptr) w.load(weight, z.D, t);
        if (bias != nullptr) b.load(bias, z.D, t);
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v.v[k][i] = affine(centred(v.v[k][i], s.mean, z.layer) * s.rstd, weight != nullptr, w.v[k][i],
                                   bias != nullptr, b.v[k][i]);
        v.store(y + at, z.D, t);
        if (t == 0) {
            if (stats != nullptr) *reinterpret_cast<float4*>(stats + 4 * n) = make_float4(s.mean, s.rstd, sf.mean, sf.rstd);
            if (flag != nullptr && !(s.rstd > 0.0f && (!POST || sf.rstd > 0.0f))) report(flag, op_id);
        }
    }
}

// Where the sums over rows go: a partial's D values at part[slot][partial], null where not wanted.
enum { W, B, PW, PB, GATE, SUMS };
struct Parts {
    float* part[SUMS];
};

template <int WAVES, int NK, bool POST, bool GATED>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES, WAVES == 1 ? 2 : 4)
norm_backward(Sizes z, Partition pt, const float* __restrict__ dr, const float* __restrict__ dy,
              const float* __restrict__ r, const float* __restrict__ f, const float* __restrict__ gate,
              const float* __restrict__ post_weight, const float* __restrict__ post_bias,
              const float* __restrict__ weight, const float* __restrict__ stats, float* __restrict__ dx,
              float* __restrict__ df, float* __restrict__ dgate, Parts parts, int* flag, int op_id) {
    constexpr int T = 64 * WAVES;
    using Row = Chunks<T, NK>;
    __shared__ float lds[WAVES == 1 ? 4 * T * NK * 4 : RowSum<WAVES, NK>::LDS];
    const int t = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int sub = WAVES == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    RowSum<WAVES, NK> sum{lds, t, z.D, 0};
    const long long section = blockIdx.x / pt.partials, p_in = blockIdx.x % pt.partials;
    const long long first = (p_in * pt.join + sub) * pt.rows;
    const long long end = first + pt.rows < pt.section_rows ? first + pt.rows : pt.section_rows;
    Row acc[SUMS];
#pragma unroll
    for (int q = 0; q < SUMS; ++q) acc[q].clear();
    // Where four values a thread make a row, its weights stay in registers and the next row's values are in
    // flight while a row is worked on.
    constexpr bool AHEAD = WAVES > 1 && NK == 1;
    Row next_r, next_dy, next_dr, next_f, held_w, held_pw, held_pb;
    float4 next_st;
    const auto fetch = [&](long long k0) {
        if (k0 >= end) return;
        const long long n = section * pt.section_rows + k0;
        const size_t at = (size_t)n * z.D;
        next_st = *reinterpret_cast<const float4*>(stats + 4 * n);
        next_r.load(r + at, z.D, t);
        if (dy != nullptr) next_dy.load(dy + at, z.D, t);
        if (dr != nullptr) next_dr.load(dr + at, z.D, t);
        if (f != nullptr) next_f.load(f + at, z.D, t);
    };
    if (AHEAD) {
        fetch(first);
        if (weight != nullptr) held_w.load(weight, z.D, t);
        if (POST && post_weight != nullptr) held_pw.load(post_weight, z.D, t);
        if (POST && GATED && post_bias != nullptr) held_pb.load(post_bias, z.D, t);
    }
    for (long long k0 = first; k0 < end; ++k0) {
        const long long n = section * pt.section_rows + k0;
        const size_t at = (size_t)n * z.D;
        if (!AHEAD) fetch(k0);
        const float4 st = next_st;
        Row hat = next_r, a = next_dy, d = next_dr, u = next_f, w = held_w;
        if (AHEAD) fetch(k0 + 1);
        if (dy != nullptr) {
            if (!AHEAD && weight != nullptr) w.load(weight, z.D, t);
#pragma unroll
            for (int k = 0; k < NK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    hat.v[k][i] = centred(hat.v[k][i], st.x, z.layer) * st.y;
                    acc[W].v[k][i] = acc[W].v[k][i] + a.v[k][i] * hat.v[k][i];
                    acc[B].v[k][i] = acc[B].v[k][i] + a.v[k][i];
                    if (weight != nullptr) a.v[k][i] = a.v[k][i] * w.v[k][i];
                }
            float c1 = 0.0f, c2;
            const auto plain = [&](int k, int i) { return a.v[k][i]; };
            const auto product = [&](int k, int i) { return a.v[k][i] * hat.v[k][i]; };
            if (z.layer) {
                sum.two(plain, product, c1, c2);
                c1 = mean_of(c1, z.D);
            } else {
                c2 = sum.one(product);
            }
            c2 = mean_of(c2, z.D);
#pragma unroll
            for (int k = 0; k < NK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float b = backward(a.v[k][i], hat.v[k][i], st.y, c1, c2, z.layer);
                    d.v[k][i] = dr != nullptr ? d.v[k][i] + b : b;
                }
        }
        if (dx != nullptr) d.store(dx + at, z.D, t);
        if (flag != nullptr) {
            bool bad = false;
#pragma unroll
            for (int k = 0; k < NK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    bad = bad || (4 * (t + T * k) + i < z.D && !__builtin_isfinite(d.v[k][i]));
            if (bad) report(flag, op_id);
        }
        if (f == nullptr) continue;
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) d.v[k][i] = d.v[k][i] * z.scale;
        if constexpr (POST) {  // hat: f normalised
#pragma unroll
            for (int k = 0; k < NK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) hat.v[k][i] = centred(u.v[k][i], st.z, z.layer) * st.w;
            if (AHEAD) w = held_pw;
            else if (post_weight != nullptr) w.load(post_weight, z.D, t);
            if (GATED) {
                Row b = held_pb;
                if (!AHEAD && post_bias != nullptr) b.load(post_bias, z.D, t);
#pragma unroll
                for (int k = 0; k < NK; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        u.v[k][i] = affine(hat.v[k][i], post_weight != nullptr, w.v[k][i], post_bias != nullptr, b.v[k][i]);
            }
        }
        if constexpr (GATED) {
            const long long row = n / pt.group_rows;
            Row g;
            g.load(gate + (size_t)row * z.D, z.D, t);
#pragma unroll
            for (int k = 0; k < NK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    acc[GATE].v[k][i] = acc[GATE].v[k][i] + d.v[k][i] * u.v[k][i];
                    d.v[k][i] = d.v[k][i] * g.v[k][i];
                }
            if (pt.gate_inside && (k0 + 1) % pt.group_rows == 0) {  // the group is whole
                if (dgate != nullptr) acc[GATE].store(dgate + (size_t)row * z.D, z.D, t);
                acc[GATE].clear();
            }
        }
        if constexpr (POST) {
#pragma unroll
            for (int k = 0; k < NK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    acc[PW].v[k][i] = acc[PW].v[k][i] + d.v[k][i] * hat.v[k][i];
                    acc[PB].v[k][i] = acc[PB].v[k][i] + d.v[k][i];
                    if (post_weight != nullptr) d.v[k][i] = d.v[k][i] * w.v[k][i];
                }
            float c1 = 0.0f, c2;
            const auto plain = [&](int k, int i) { return d.v[k][i]; };
            const auto product = [&](int k, int i) { return d.v[k][i] * hat.v[k][i]; };
            if (z.layer) {
                sum.two(plain, product, c1, c2);
                c1 = mean_of(c1, z.D);
            } else {
                c2 = sum.one(product);
            }
            c2 = mean_of(c2, z.D);
#pragma unroll
            for (int k = 0; k < NK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) d.v[k][i] = backward(d.v[k][i], hat.v[k][i], st.w, c1, c2, z.layer);
        }
        if (df != nullptr) d.store(df + at, z.D, t);
    }
#pragma unroll
    for (int q = 0; q < SUMS; ++q) {
        if ((q == PW || q == PB) && !POST) continue;
        if (q == GATE && !GATED) continue;
        float* out = parts.part[q];
        if (out == nullptr) continue;
        out += (size_t)blockIdx.x * z.D;
        if constexpr (WAVES == 1) {
            // the four strands' values at [strand][k][lane][4]
            __syncthreads();
            float4* p = reinterpret_cast<float4*>(lds);
#pragma unroll
            for (int k = 0; k < NK; ++k)
                p[(sub * NK + k) * 64 + t] = make_float4(acc[q].v[k][0], acc[q].v[k][1], acc[q].v[k][2], acc[q].v[k][3]);
            __syncthreads();
            const int k = threadIdx.x >> 6;
            if (k < NK) {
                float4 v[4];
#pragma unroll
                for (int s = 0; s < 4; ++s) v[s] = p[(s * NK + k) * 64 + t];
                const float o[4] = {(v[0].x + v[1].x) + (v[2].x + v[3].x), (v[0].y + v[1].y) + (v[2].y + v[3].y),
                                    (v[0].z + v[1].z) + (v[2].z + v[3].z), (v[0].w + v[1].w) + (v[2].w + v[3].w)};
                const int at = 4 * (t + T * k);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at + i < z.D) out[at + i] = o[i];
            }
        } else {
            acc[q].store(out, z.D, t);
        }
    }
}

// out[j][i] = the sum of P partials' column i: a block takes 64 columns of one sum j, its wavefront h the partials
// p with p mod 16 = h.
struct Totals {
    const float* part[4 + 1];
    float* out[4 + 1];
    long long partials[4 + 1];
    int sums;          // of them; the last may be the gate's, which repeats
    long long repeat;  // the last one's results, `partials` apart
};

__global__ void __launch_bounds__(1024)
norm_totals(Totals z, int D) {
    __shared__ float lds[16][64];
    const int lane = threadIdx.x & 63, h = threadIdx.x >> 6;
    const int i = blockIdx.x * 64 + lane;
    const int j = blockIdx.y, q = j < z.sums ? j : z.sums - 1;
    const long long again = j - q, P = z.partials[q];
    const float* __restrict__ p = z.part[q] + again * P * D;
    float s = 0.0f;
    if (i < D) {
#pragma unroll 8
        for (long long k = h; k < P; k += 16) s = s + p[k * D + i];
    }
    lds[h][lane] = s;
    __syncthreads();
    if (h == 0 && i < D) {
        float v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = lds[k][lane];
#pragma unroll
        for (int n = 8; n > 0; n /= 2)
#pragma unroll
            for (int k = 0; k < n; ++k) v[k] = v[2 * k] + v[2 * k + 1];
        z.out[q][again * D + i] = v[0];
    }
}

bool sizes_ok(const rg_norm_config* c) {
    return c != nullptr && c->N >= 0 && c->D >= 1 && c->D <= RG_NORM_MAX_D && c->eps >= 0.0f && c->gate_rows >= 0 &&
           (c->gate_rows == 0 || (c->gate_rows <= c->N && c->N % c->gate_rows == 0));
}

Sizes sizes_of(const rg_norm_config* c) { return Sizes{c->N, c->D, c->eps, c->scale, c->rms == 0}; }

// Blocks of a forward launch whose rows take a block each: two a compute unit, each with a row ahead.
constexpr long long FORWARD_BLOCKS = 512;

// run(WAVES, NK) with the values that hold a row of D. Rows of 2049 to 4096 values take eight wavefronts in the
// forward pass (sixteen wait for each other at its barriers: 4096 rows of 4096 59 -> 82 us) and sixteen
// in the backward pass, whose sums over rows would not leave registers for two rows otherwise.
template <bool FORWARD, class F>
void with_row(int D, F run) {
    using std::integral_constant;
    const auto of = [&](auto waves, auto nk) { run(waves, nk); };
    constexpr integral_constant<int, 1> one;
    constexpr integral_constant<int, 2> two;
    constexpr integral_constant<int, 3> three;
    constexpr integral_constant<int, 4> four;
    constexpr integral_constant<int, 8> eight;
    constexpr integral_constant<int, 16> sixteen;
    if (D <= 256) of(one, one);
    else if (D <= 512) of(one, two);
    else if (D <= 768) of(one, three);
    else if (D <= 1024) of(one, four);
    else if (D <= 2048) of(eight, one);
    else if (D <= 4096) {
        if constexpr (FORWARD) of(eight, two);
        else of(sixteen, one);
    } else if (D <= 8192) of(sixteen, two);
    else of(sixteen, four);
}

}  // namespace
}  // namespace rg

extern "C" {

void rg_norm_config_init(rg_norm_config* cfg) {
    if (!cfg) return;
    cfg->N = 0;
    cfg->D = 0;
    cfg->rms = 0;
    cfg->post = 0;
    cfg->gate_rows = 0;
    cfg->eps = 1e-5f;
    cfg->scale = 1.0f;
}

int rg_residual_norm_fp32(const rg_norm_config* cfg, const float* x, const float* f, const float* gate,
                          const float* post_weight, const float* post_bias, const float* weight,
                          const float* bias, float* r, float* y, float* stats, int* flag, int op_id,
                          void* stream) {
    using namespace rg;
    if (!sizes_ok(cfg)) return hipErrorInvalidValue;
    if (cfg->N == 0) return hipSuccess;
    if (!x || !y || !f != !r || (!f && (cfg->post || cfg->gate_rows || gate)) || !gate != (cfg->gate_rows == 0) ||
        (!cfg->post && (post_weight || post_bias)) || (reinterpret_cast<uintptr_t>(stats) & 15) != 0)
        return hipErrorInvalidValue;
    const Sizes z = sizes_of(cfg);
    const long long group = cfg->gate_rows > 0 ? cfg->N / cfg->gate_rows : 1;
    with_row<true>(cfg->D, [&](auto waves, auto nk) {
        constexpr int WV = decltype(waves)::value, NK = decltype(nk)::value;
        constexpr int rows = WV == 1 ? 4 : 1;
        const long long needed = (cfg->N + rows - 1) / rows;
        const long long most = WV == 1 ? 1 << 20 : FORWARD_BLOCKS;
        const dim3 grid((unsigned)(needed < most ? needed : most)), block(WV == 1 ? 256 : 64 * WV);
        auto kernel = cfg->post ? norm_forward<WV, NK, true> : norm_forward<WV, NK, false>;
        hipLaunchKernelGGL(kernel, grid, block, 0, static_cast<hipStream_t>(stream), z, group, x, f, gate, post_weight,
                           post_bias, weight, bias, r, y, stats, flag, op_id);
    });
    return hipGetLastError();
}

int rg_residual_norm_grad_workspace(const rg_norm_config* cfg, int sums, size_t* bytes) {
    if (!rg::sizes_ok(cfg) || !bytes) return hipErrorInvalidValue;
    if (cfg->N == 0 || !sums) {
        *bytes = 0;
        return hipSuccess;
    }
    const rg::Partition pt = repro_norm::partition(cfg->N, cfg->D, cfg->gate_rows);
    *bytes = (size_t)rg::SUMS * pt.sections * pt.partials * cfg->D * sizeof(float);
    return hipSuccess;
}

int rg_residual_norm_grad_fp32(const rg_norm_config* cfg, const float* dr, const float* dy, const float* r,
                               const float* f, const float* gate, const float* post_weight,
                               const float* post_bias, const float* weight, const float* stats, float* dx,
                               float* df, float* dgate, float* dpost_weight, float* dpost_bias,
                               float* dweight, float* dbias, void* workspace, size_t workspace_bytes,
                               int* flag, int op_id, void* stream) {
    using namespace rg;
    if (!sizes_ok(cfg)) return hipErrorInvalidValue;
    if (cfg->N == 0) return hipSuccess;
    if ((!dr && !dy) || !r || !stats || (reinterpret_cast<uintptr_t>(stats) & 15) != 0 ||
        (!f && (cfg->post || cfg->gate_rows || df)) || !gate != (cfg->gate_rows == 0) || (dgate && !gate) ||
        (!cfg->post && (post_weight || post_bias || dpost_weight || dpost_bias)) || (!dy && (dweight || dbias)))
        return hipErrorInvalidValue;
    const Partition pt = repro_norm::partition(cfg->N, cfg->D, cfg->gate_rows);
    const long long P = pt.sections * pt.partials;
    float* out[SUMS] = {dweight, dbias, dpost_weight, dpost_bias, pt.gate_inside ? nullptr : dgate};
    bool any = false;
    for (float* o : out) any = any || o;
    size_t needed = 0;
    (void)rg_residual_norm_grad_workspace(cfg, any ? 1 : 0, &needed);
    if (needed > 0 && (!workspace || workspace_bytes < needed || (reinterpret_cast<uintptr_t>(workspace) & 3) != 0))
        return hipErrorInvalidValue;
    Parts parts;
    Totals totals;
    totals.sums = 0;
    totals.repeat = 1;
    for (int q = 0; q < SUMS; ++q) {
        parts.part[q] = out[q] ? static_cast<float*>(workspace) + (size_t)q * P * cfg->D : nullptr;
        if (!out[q]) continue;
        totals.part[totals.sums] = parts.part[q];
        totals.out[totals.sums] = out[q];
        totals.partials[totals.sums++] = q == GATE ? pt.partials : P;
        if (q == GATE) totals.repeat = pt.sections;
    }
    const Sizes z = sizes_of(cfg);
    hipStream_t st = static_cast<hipStream_t>(stream);
    with_row<false>(cfg->D, [&](auto waves, auto nk) {
        constexpr int WV = decltype(waves)::value, NK = decltype(nk)::value;
        auto kernel = cfg->post ? (gate ? norm_backward<WV, NK, true, true> : norm_backward<WV, NK, true, false>)
                                : (gate ? norm_backward<WV, NK, false, true> : norm_backward<WV, NK, false, false>);
        hipLaunchKernelGGL(kernel, dim3((unsigned)P), dim3(WV == 1 ? 256 : 64 * WV), 0, st, z, pt, dr, dy, r, f, gate,
                           post_weight, post_bias, weight, stats, dx, df, dgate, parts, flag, op_id);
    });
    int rc = hipGetLastError();
    if (rc == hipSuccess && totals.sums > 0) {
        // (The partition has at most 4096 partials and 2048 sections.)
        hipLaunchKernelGGL(norm_totals, dim3((cfg->D + 63) / 64, (unsigned)(totals.sums - 1 + totals.repeat)), dim3(1024), 0,
                           st, totals, cfg->D);
        rc = hipGetLastError();
    }
    return rc;
}

}  // extern "C"
