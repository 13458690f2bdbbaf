// The attention's gradients on the matrix cores.
//
// A block takes 128 keys of a head, 32 a wavefront, and goes through the queries 32 at a time, which its wavefronts share in LDS:
// S = Q K^T and dP = dY V^T with queries as rows (row 8 g + 4 h + r is query 8 g + 2 r + h, as in the forward pass), so a
// register of P or dS is the operand of dV^T = dY^T P and dK^T = Q^T dS for two successive queries. K and V stay in registers, as
// the operands of the first two, and K in LDS for dQ = dS K, which needs dS along its rows: it goes through LDS, and the wavefronts
// share the tile's 32 rows of dQ by 16 x 16 blocks over all 128 keys (v_mfma_f32_16x16x4_f32: four products in ascending order).
//
// dQ's sum over key blocks is taken from what each block leaves (no atomics, whose order would vary): 4 D bytes a query and
// block written and read beside the 5 x 128 x D multiply-adds that make them. Sums of chunks of 256 queries go to dK
// and dV as they are done, or stay apart where the queries are split over blocks.
//
// As in the forward pass vector instructions add to the products' time (about a sixth of it). Loads go by buffer offsets without
// branches: with branches each waited for the one before, and the pass of 2 x 16 heads of 4096 x 4096 x 64 took 4.75 ms
// where it takes 3.17 (108 TFLOP/s). Two blocks a compute unit up to 64 values a head, whose registers hold two wavefronts a
// SIMD.
#include "rg_attention.h"

namespace rg {
namespace attention {
namespace {

typedef float Block16 __attribute__((ext_vector_type(16)));
typedef float Block4 __attribute__((ext_vector_type(4)));

constexpr int STEP = 32;                              // queries at a time
constexpr int DIAGONALS = KEY_BLOCK + QUERY_CHUNK;    // distances of a block and chunk, one more than there are
constexpr int DS_STRIDE = KEY_BLOCK + STEP + 1;     // a row of dS and zeros, over which a diagonal goes on into its neighbours

__device__ __forceinline__ Block16 zero16() {
    Block16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.0f;
    return z;
}
__device__ __forceinline__ Block16 mfma(float a, float b, Block16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}
// Keeps the compiler from fetching operands of later products early, which takes registers that there are not.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }
// A value that the compiler does not compute addresses from ahead of a loop.
__device__ __forceinline__ int fresh(int v) {
    asm volatile("" : "+v"(v));
    return v;
}
__device__ __forceinline__ Block4 mfma4(float a, float b, Block4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float part_of(const float4& v, int r) { return r == 0 ? v.x : r == 1 ? v.y : r == 2 ? v.z : v.w; }

// Where a block and chunk are, and what they leave. Key blocks first .. first + count of the `blocks`.
struct Work {
    int first, count, chunks, parts, a_part;
    int direct;                 // dk and dv are the results themselves, [B][Tk][KVH][D], else [chunk or 1][B][H][Tk][D]
    float *dk, *dv;
    float* dq;                  // [count][B][H][Tq][D]
    float* diagonals;           // [B][H][count][chunks][DIAGONALS], or null
    int* broken;                // a number for each block: whether `repair` has to redo it; null where it never has to
};
struct Place {
    int bh, slot, part;
};
__device__ __forceinline__ Place place_of(const Problem& z, const Work& w) {
    const int heads = z.B * z.H, rest = (int)(blockIdx.x / heads);
    return Place{(int)(blockIdx.x % heads), rest / w.parts, rest % w.parts};
}
// Where a key's sums of a chunk go: the chunk's own place, or the one that all chunks are added to.
__device__ __forceinline__ size_t out_of(const Problem& z, const Work& w, int bh, int chunk) {
    return w.direct ? ((size_t)(bh / z.H) * z.Tk * z.KVH + bh % z.H) * z.D
                    : ((size_t)(w.parts > 1 ? chunk : 0) * z.B * z.H + bh) * z.Tk * z.D;
}

__device__ __forceinline__ int last_end(const Problem& z, int len, int i) {
    return z.causal ? max(0, min(len, i + z.start + 1)) : len;
}
// Whether a key block's keys are seen by a query before `rows` (the mask aside).
__device__ __forceinline__ bool live(const Problem& z, int len, int block, int rows) {
    return block * KEY_BLOCK < last_end(z, len, min(rows, z.Tq) - 1);
}

// Without a bias and dropout heads of up to 32 values leave room for a third wavefront a SIMD (4 x 16 heads of 2048 x 2048 x 32: 880 us, with two
// 901; 8 x 12 of 1024 x 1024 x 16: 321, 364).
template <int DB, bool BIAS, bool DROP, bool QUADS>
__global__ void __launch_bounds__(256, DB == 1 && !BIAS && !DROP ? 3 : 2)
backward_tiles(Problem z, Gradients g, Work w) {
    constexpr int DP = 32 * DB, QS = DP + 4, KS = DP + 8;
    __shared__ float Ks[KEY_BLOCK * KS], Qs[STEP * QS], Ys[STEP * QS], Ds_[STEP + STEP * DS_STRIDE];
    __shared__ float Bs[BIAS ? 160 : 1], Sums[BIAS ? DIAGONALS : 1];
    __shared__ float4 Query[(BIAS ? 1 : 2) * STEP];  // m, 1 / L, delta, and the keys that the query sees, as bits; the same with m = 0
    __shared__ uint32_t Masks[STEP][4];
    float* Ds = Ds_ + STEP;  // (zeros before the first row, too)
    const uint64_t seed = z.seed_at ? *z.seed_at : z.seed;
    const int t = threadIdx.x, lane = t & 63, col = lane & 31, half = lane >> 5, wave = t >> 6;
    const Place at = place_of(z, w);
    const int bh = at.bh, b = bh / z.H, h = bh % z.H, slot = at.slot, heads = z.B * z.H;
    const int block = w.first + slot, k0 = block * KEY_BLOCK;
    const int len = keys_of(z, b), key = k0 + 32 * wave + col;
    const size_t row0 = (size_t)bh * z.Tq;
    const size_t out_stride = (size_t)(w.direct ? z.KVH : 1) * z.D;

    if (!live(z, len, block, z.Tq)) {
        const size_t out = out_of(z, w, bh, 0);
        if (w.direct)
            for (int n = t; n < KEY_BLOCK * z.D; n += 256)
                if (k0 + n / z.D < z.Tk) {
                    w.dk[out + (k0 + n / z.D) * out_stride + n % z.D] = 0.0f;
                    w.dv[out + (k0 + n / z.D) * out_stride + n % z.D] = 0.0f;
                }
        if (w.broken && t == 0) w.broken[blockIdx.x] = 0;
        return;
    }

    float k[16 * DB], v[16 * DB];  // value 2 n + half of the lane's key
    float broken = 0.0f;
    // a thread brings four values in each 32 of a row
    const int lrow = t >> 3, lcol = 4 * (t & 7);
    const auto keys_to_lds = [&](const float* base, long long stride) {
        const Rows rows = rows_at(base + k0 * stride, min(KEY_BLOCK, len - k0), stride, z.D);
        const uint32_t at = ((uint32_t)lrow * (uint32_t)stride + lcol) * 4;
        float4 x[4 * DB];
#pragma unroll
        for (int n = 0; n < 4 * DB; ++n)
            x[n] = four<QUADS>(rows, at + 128 * (n % DB) + n / DB * 128 * (uint32_t)stride, z.D - lcol - 32 * (n % DB));
#pragma unroll
        for (int n = 0; n < 4 * DB; ++n) *reinterpret_cast<float4*>(Ks + (lrow + n / DB * 32) * KS + lcol + 32 * (n % DB)) = x[n];
    };
    const auto take = [&](float* to) {
#pragma unroll
        for (int n = 0; n < 8 * DB; ++n) {
            const float4 x = *reinterpret_cast<const float4*>(Ks + (32 * wave + col) * KS + 4 * n);
            to[2 * n] = half ? x.y : x.x;
            to[2 * n + 1] = half ? x.w : x.z;
        }
    };
    for (int n = t; n < STEP; n += 256) Ds_[n] = 0.0f;
    for (int n = t; n < STEP * (STEP + 1); n += 256) Ds[n / (STEP + 1) * DS_STRIDE + KEY_BLOCK + n % (STEP + 1)] = 0.0f;
    keys_to_lds(value_at(z, b, h, 0), z.v_stride[1]);
    __syncthreads();
    take(v);
    __syncthreads();
    keys_to_lds(key_at(z, b, h, 0), z.k_stride[1]);
    __syncthreads();
    take(k);
#pragma unroll
    for (int n = 0; n < 16 * DB; ++n) {
        broken = __builtin_fmaf(k[n], 0.0f, broken);
        k[n] = z.flip ? -k[n] : k[n];
    }

    const float* qbase = query_at(z, b, h, 0);
    const float* ybase = g.dy + ((size_t)b * z.Tq * z.H + h) * z.D;
    const int ystride = z.H * z.D;
    float4 qn[DB], yn[DB];
    float bn = 0.0f;
    float2 sn;
    float en;
    uint32_t mn = ~0u;
    const auto load = [&](int i0) {
        const int t = fresh(threadIdx.x), lrow = t >> 3, lcol = 4 * (t & 7);
        const uint32_t qat = ((uint32_t)lrow * (uint32_t)z.q_stride[1] + lcol) * 4, yat = ((uint32_t)lrow * (uint32_t)ystride + lcol) * 4;
        const Rows qr = rows_at(qbase + i0 * z.q_stride[1], min(STEP, z.Tq - i0), z.q_stride[1], z.D);
        const Rows yr = rows_at(ybase + (long long)i0 * ystride, min(STEP, z.Tq - i0), ystride, z.D);
#pragma unroll
        for (int x = 0; x < DB; ++x) {
            const int left = x < DB - 1 ? 4 : z.D - lcol - 32 * x;
            qn[x] = four<QUADS>(qr, qat + 128 * x, left);
            yn[x] = four<QUADS>(yr, yat + 128 * x, left);
        }
        const size_t row = row0 + min(i0 + (t & (STEP - 1)), z.Tq - 1);
        sn = reinterpret_cast<const float2*>(g.stats)[row];
        en = g.delta[row];
        if (z.mask) {
            const int i = min(i0 + ((t >> 2) & (STEP - 1)), z.Tq - 1), word = min(k0 / 32 + (t & 3), (z.Tk - 1) / 32);
            const unsigned long long* m = z.mask + b * z.mask_stride[0] + h * z.mask_stride[1] + i * z.mask_stride[2];
            mn = reinterpret_cast<const uint32_t*>(m)[word];
        }
        if (BIAS) {
            const int c = k0 + t - (STEP - 1) - i0 + z.Tq - 1;  // (outside of the bias no pair needs it)
            bn = z.bias[(size_t)h * (z.Tq + z.Tk - 1) + max(0, min(c, z.Tq + z.Tk - 2))];
        }
    };
    const auto store = [&](int i0) {
        const int t = fresh(threadIdx.x), lrow = t >> 3, lcol = 4 * (t & 7);
#pragma unroll
        for (int x = 0; x < DB; ++x) {
            const int d = lcol + 32 * x, to = lrow * QS + (d & ~7) + (d & 4) / 2;  // values 2 r + h of eight at 4 h + r
            *reinterpret_cast<float2*>(Qs + to) = make_float2(qn[x].x, qn[x].z);
            *reinterpret_cast<float2*>(Qs + to + 4) = make_float2(qn[x].y, qn[x].w);
            *reinterpret_cast<float2*>(Ys + to) = make_float2(yn[x].x, yn[x].z);
            *reinterpret_cast<float2*>(Ys + to + 4) = make_float2(yn[x].y, yn[x].w);
        }
        if (t < (BIAS ? 1 : 2) * STEP) {
            const int i = i0 + (t & (STEP - 1));
            Query[t] = make_float4(t < STEP ? sn.x : 0.0f, sn.y, en, __int_as_float(i < z.Tq ? last_end(z, len, i) : 0));
        }
        if (t >= 128) Masks[(t >> 2) & (STEP - 1)][t & 3] = mn;
        if (BIAS && t < KEY_BLOCK + STEP - 1) Bs[t] = bias_term(bn);
    };
    const int row_of = (col & 24) + 2 * (col & 3) + ((col >> 2) & 1);     // the query that row `col` of an operand is
    const int place_in = (col & 24) + 4 * (col & 1) + ((col >> 1) & 3);   // where value `col` of 32 is in Qs and Ys
    const int first_chunk = at.part * w.a_part, last_chunk = min(w.chunks, first_chunk + w.a_part);
    bool begun = false;
    for (int chunk = first_chunk; chunk < last_chunk; ++chunk) {
        const int c0 = chunk * QUERY_CHUNK, c1 = min(c0 + QUERY_CHUNK, z.Tq);
        if (!live(z, len, block, c1)) continue;
        float* diagonals = BIAS && w.diagonals ? w.diagonals + (((size_t)bh * w.count + slot) * w.chunks + chunk) * DIAGONALS : nullptr;
        Block16 dk[DB], dv[DB];
#pragma unroll
        for (int n = 0; n < DB; ++n) dk[n] = dv[n] = zero16();
        int i0 = c0;
        while (!live(z, len, block, i0 + STEP)) i0 += STEP;  // (the chunk's last step is live)
        __syncthreads();
        load(i0);
        store(i0);
        if (BIAS)
            for (int n = t; n < DIAGONALS; n += 256) Sums[n] = 0.0f;
        lds_barrier();
        for (; i0 < c1; i0 += STEP) {
            const bool more = i0 + STEP < c1;
            Block16 s = zero16(), dp = zero16();
            {
                const float* qs = Qs + row_of * QS + 4 * half;
                const float* ys = Ys + row_of * QS + 4 * half;
                float4 a = *reinterpret_cast<const float4*>(qs), c = *reinterpret_cast<const float4*>(ys);
#pragma unroll
                for (int u = 0; u < 4 * DB; ++u) {
                    const int ahead = u + 1 < 4 * DB ? u + 1 : u;
                    const float4 an = *reinterpret_cast<const float4*>(qs + 8 * ahead);
                    const float4 cn = *reinterpret_cast<const float4*>(ys + 8 * ahead);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s = mfma(part_of(a, r), k[4 * u + r], s);
                        dp = mfma(part_of(c, r), v[4 * u + r], dp);
                    }
                    a = an;
                    c = cn;
                    fence();
                }
            }
            uint32_t keep[4];
            if (DROP) {
                // a call's four words are four keys', neighbours in a quad of lanes: each makes those of another query
                uint32_t bits = 0;
                const int r = lane & 3;
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const auto x = repro_dropout::pair_words((uint32_t)(key >> 2), i0 + 8 * n + 2 * r + half, bh, seed);
#pragma unroll
                    for (int q = 0; q < 4; ++q) bits |= (uint32_t)(x.w[q] >= z.threshold) << (4 * n + q);
                }
                keep[0] = __builtin_amdgcn_update_dpp(0, bits, 0x00, 0xF, 0xF, true) >> r;
                keep[1] = __builtin_amdgcn_update_dpp(0, bits, 0x55, 0xF, 0xF, true) >> r;
                keep[2] = __builtin_amdgcn_update_dpp(0, bits, 0xAA, 0xF, 0xF, true) >> r;
                keep[3] = __builtin_amdgcn_update_dpp(0, bits, 0xFF, 0xF, 0xF, true) >> r;
            }
            const bool large = !BIAS && __any(is_large(Query[lane & (STEP - 1)].x));
            if (large) {  // the exponents are made here, and kept by what follows
#pragma unroll
                for (int n = 0; n < 16; ++n)
                    s[n] = repro_attention::less(s[n], s[n] * z.factor, z.factor, Query[8 * (n / 4) + 2 * (n % 4) + half].x, false);
            }
            const float factor = large ? 1.0f : z.factor;
            const float4* rows = Query + (large ? STEP : 0);
            const auto differentials = [&](auto edge) {
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                    const int q = 8 * (n / 4) + 2 * (n % 4) + half;
                    const float4 row = rows[q];
                    const float x = BIAS ? __builtin_fmaf(s[n], z.factor, Bs[32 * wave + col - q + STEP - 1]) - row.x
                                         : __builtin_fmaf(s[n], factor, -row.x);
                    float p = e2(x) * row.y, d = dp[n], u = p;
                    if (DROP) {
                        const bool kept = (keep[n % 4] >> (4 * (n / 4)) & 1) != 0;
                        u = kept ? p * z.keep_factor : 0.0f;
                        d = kept ? d * z.keep_factor : 0.0f;
                    }
                    d = ds_of(p, d, row.z);
                    if (decltype(edge)::value) {
                        const bool see = (int)(key < __float_as_int(row.w)) & (int)(Masks[q][wave] >> col & 1);
                        u = see ? u : 0.0f;
                        d = see ? d : 0.0f;
                    }
                    s[n] = u;
                    dp[n] = d;
                    Ds[q * DS_STRIDE + 32 * wave + col] = d;
                    if (n % 4 == 3) fence();
                }
            };
            // whether every pair of the wavefront's is seen
            if (!z.mask && i0 + STEP <= z.Tq && k0 + 32 * wave + 32 <= last_end(z, len, i0)) differentials(std::false_type());
            else differentials(std::true_type());
            {
                const float* qs = Qs + half * QS + place_in;
                const float* ys = Ys + half * QS + place_in;
                float a[DB], c[DB];
#pragma unroll
                for (int x = 0; x < DB; ++x) a[x] = ys[32 * x], c[x] = qs[32 * x];
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                    const int m = n < 15 ? n + 1 : n, ahead = (8 * (m / 4) + 2 * (m % 4)) * QS;
                    float an[DB], cn[DB];
#pragma unroll
                    for (int x = 0; x < DB; ++x) an[x] = ys[ahead + 32 * x], cn[x] = qs[ahead + 32 * x];
#pragma unroll
                    for (int x = 0; x < DB; ++x) {
                        dv[x] = mfma(a[x], s[n], dv[x]);
                        dk[x] = mfma(c[x], dp[n], dk[x]);
                    }
#pragma unroll
                    for (int x = 0; x < DB; ++x) a[x] = an[x], c[x] = cn[x];
                    fence();
                }
            }
            lds_barrier();
            if (more) load(i0 + STEP);  // (in flight under dQ's products)
            {
                const int c16 = lane & 15, group = lane >> 4, q0 = 16 * (wave & 1), d0 = 16 * DB * (wave >> 1);
                Block4 dq[DB];
#pragma unroll
                for (int x = 0; x < DB; ++x) dq[x] = Block4{0.0f, 0.0f, 0.0f, 0.0f};
                const float* ds = Ds + (q0 + c16) * DS_STRIDE + group;
                const float* ks = Ks + group * KS + d0 + c16;
                float a[4], c[4][DB];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    a[r] = ds[4 * r];
#pragma unroll
                    for (int x = 0; x < DB; ++x) c[r][x] = ks[4 * r * KS + 16 * x];
                }
#pragma unroll
                for (int n = 0; n < KEY_BLOCK / 16; ++n) {
                    const int ahead = 16 * (n + 1 < KEY_BLOCK / 16 ? n + 1 : n);
                    float an[4], cn[4][DB];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        an[r] = ds[ahead + 4 * r];
#pragma unroll
                        for (int x = 0; x < DB; ++x) cn[r][x] = ks[(ahead + 4 * r) * KS + 16 * x];
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int x = 0; x < DB; ++x) dq[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], c[r][x], dq[x], 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        a[r] = an[r];
#pragma unroll
                        for (int x = 0; x < DB; ++x) c[r][x] = cn[r][x];
                    }
                    fence();
                }
                const Rows rows = rows_at(w.dq + ((size_t)slot * heads * z.Tq + row0 + i0) * z.D, min(STEP, z.Tq - i0), z.D, z.D);
                const int from = fresh(lane);
#pragma unroll
                for (int x = 0; x < DB; ++x) {
                    const int d = d0 + 16 * x + (from & 15), group = from >> 4;
                    const uint32_t to = d < z.D ? ((uint32_t)(q0 + 4 * group) * z.D + d) * 4 : NOWHERE;
#pragma unroll
                    for (int r = 0; r < 4; ++r) put_one(rows, to + (uint32_t)(4 * r * z.D), dq[x][r]);
                }
            }
            if (BIAS && w.diagonals && t < KEY_BLOCK + STEP - 1) {
                float* sum = Sums + t - (STEP - 1) - (i0 - c0) + QUERY_CHUNK - 1;
                const float* ds = Ds + t - (STEP - 1);
                float x = *sum;
#pragma unroll
                for (int q = 0; q < STEP; ++q) x = x + ds[q * (DS_STRIDE + 1)];
                *sum = x;
            }
            if (more) store(i0 + STEP);
            lds_barrier();
        }
        const bool last = w.direct && chunk == w.chunks - 1;
        const size_t chunk_out = out_of(z, w, bh, chunk);
        const bool add = w.parts == 1 && begun;
        begun = true;
        const auto leave = [&](float* base, const Block16* sum, float scale) {
            const Rows rows = rows_at(base + chunk_out + k0 * out_stride, min(KEY_BLOCK, z.Tk - k0), out_stride, z.D);
            const int lane = fresh(threadIdx.x) & 63, half = lane >> 5;
            const uint32_t to = ((uint32_t)(32 * wave + (lane & 31)) * (uint32_t)out_stride + 4 * half) * 4;
            float4 held[4 * DB];
            if (add) {
#pragma unroll
                for (int n = 0; n < 4 * DB; ++n) held[n] = four<QUADS>(rows, to + 32 * n, z.D - 8 * n - 4 * half);
            }
#pragma unroll
            for (int n = 0; n < 4 * DB; ++n) {
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    v[r] = sum[n / 4][4 * (n % 4) + r];
                    if (add) v[r] = part_of(held[n], r) + v[r];
                    if (last) v[r] = v[r] * scale + 0.0f;
                }
                put_four<QUADS>(rows, to + 32 * n, z.D - 8 * n - 4 * half, v);
            }
        };
#pragma unroll
        for (int n = 0; n < 16 * DB; ++n) {
            broken = __builtin_fmaf(dk[n / 16][n % 16], 0.0f, broken);
            broken = __builtin_fmaf(dv[n / 16][n % 16], 0.0f, broken);
        }
        leave(w.dk, dk, z.scale);
        leave(w.dv, dv, 1.0f);
        if (diagonals)
            for (int n = t; n < DIAGONALS; n += 256) diagonals[n] = Sums[n];
    }
    if (w.broken) {  // a NaN or infinity, which the products' zeros hand to pairs that are not seen, shows in every key's sums
        const int any = __syncthreads_or(broken != broken);
        if (t == 0) w.broken[blockIdx.x] = any;
    }
}

// The same for heads of more than 64 values, whose sums would leave one wavefront a SIMD and nothing to run while it waits at a
// barrier (2 x 16 heads of 2048 x 2048 x 128 in the kernel above: 1790 us, here 1600, 107 TFLOP/s): eight wavefronts of 16
// keys each, all products by 16 x 16 blocks (row 4 c + r of an operand is query 4 r + c, so that a register of P or dS is again the
// next operand, for four successive queries).
template <int DB, bool BIAS, bool DROP, bool QUADS>
__global__ void __launch_bounds__(512, 2)
backward_wide(Problem z, Gradients g, Work w) {
    constexpr int DP = 32 * DB, QS = DP + 4, KS = DP + 8;
    __shared__ float Ks[KEY_BLOCK * KS], Qs[STEP * QS], Ys[STEP * QS], Ds_[STEP + STEP * DS_STRIDE];
    __shared__ float Bs[BIAS ? 160 : 1], Sums[BIAS ? DIAGONALS : 1];
    __shared__ float4 Query[(BIAS ? 1 : 2) * STEP];  // m, 1 / L, delta, and the keys that the query sees, as bits; the same with m = 0
    __shared__ uint32_t Masks[STEP][4];
    float* Ds = Ds_ + STEP;  // (zeros before the first row, too)
    const uint64_t seed = z.seed_at ? *z.seed_at : z.seed;
    const int t = threadIdx.x, lane = t & 63, col = lane & 15, group = lane >> 4, wave = t >> 6;
    const Place at = place_of(z, w);
    const int bh = at.bh, b = bh / z.H, h = bh % z.H, slot = at.slot, heads = z.B * z.H;
    const int block = w.first + slot, k0 = block * KEY_BLOCK;
    const int len = keys_of(z, b), key = k0 + 16 * wave + col;
    const size_t row0 = (size_t)bh * z.Tq;
    const size_t out_stride = (size_t)(w.direct ? z.KVH : 1) * z.D;

    if (!live(z, len, block, z.Tq)) {
        const size_t out = out_of(z, w, bh, 0);
        if (w.direct)
            for (int n = t; n < KEY_BLOCK * z.D; n += 512)
                if (k0 + n / z.D < z.Tk) {
                    w.dk[out + (k0 + n / z.D) * out_stride + n % z.D] = 0.0f;
                    w.dv[out + (k0 + n / z.D) * out_stride + n % z.D] = 0.0f;
                }
        if (w.broken && t == 0) w.broken[blockIdx.x] = 0;
        return;
    }

    float k[8 * DB], v[8 * DB];  // value 4 n + group of the lane's key
    float broken = 0.0f;
    const int lrow = t >> 3, lcol = 4 * (t & 7);
    const auto keys_to_lds = [&](const float* base, long long stride) {
        const Rows rows = rows_at(base + k0 * stride, min(KEY_BLOCK, len - k0), stride, z.D);
        const uint32_t at = ((uint32_t)lrow * (uint32_t)stride + lcol) * 4;
        float4 x[2 * DB];
#pragma unroll
        for (int n = 0; n < 2 * DB; ++n)
            x[n] = four<QUADS>(rows, at + 128 * (n % DB) + n / DB * 256 * (uint32_t)stride, z.D - lcol - 32 * (n % DB));
#pragma unroll
        for (int n = 0; n < 2 * DB; ++n) *reinterpret_cast<float4*>(Ks + (lrow + n / DB * 64) * KS + lcol + 32 * (n % DB)) = x[n];
    };
    const auto take = [&](float* to) {
#pragma unroll
        for (int n = 0; n < 8 * DB; ++n) to[n] = Ks[(16 * wave + col) * KS + 4 * n + group];
    };
    for (int n = t; n < STEP; n += 512) Ds_[n] = 0.0f;
    for (int n = t; n < STEP * (STEP + 1); n += 512) Ds[n / (STEP + 1) * DS_STRIDE + KEY_BLOCK + n % (STEP + 1)] = 0.0f;
    keys_to_lds(value_at(z, b, h, 0), z.v_stride[1]);
    __syncthreads();
    take(v);
    __syncthreads();
    keys_to_lds(key_at(z, b, h, 0), z.k_stride[1]);
    __syncthreads();
    take(k);
#pragma unroll
    for (int n = 0; n < 8 * DB; ++n) {
        broken = __builtin_fmaf(k[n], 0.0f, broken);
        k[n] = z.flip ? -k[n] : k[n];
    }

    // the first four wavefronts bring the queries, the others the gradients
    const bool first_half = __builtin_amdgcn_readfirstlane(wave) < 4;
    const float* base = first_half ? query_at(z, b, h, 0) : g.dy + ((size_t)b * z.Tq * z.H + h) * z.D;
    const long long stride = first_half ? z.q_stride[1] : (long long)z.H * z.D;
    float4 qn[DB];
    float bn = 0.0f;
    float2 sn;
    float en;
    uint32_t mn = ~0u;
    const auto load = [&](int i0) {
        const int t = fresh(threadIdx.x), lrow = (t >> 3) & (STEP - 1), lcol = 4 * (t & 7);
        const uint32_t at = ((uint32_t)lrow * (uint32_t)stride + lcol) * 4;
        const Rows rows = rows_at(base + i0 * stride, min(STEP, z.Tq - i0), stride, z.D);
#pragma unroll
        for (int x = 0; x < DB; ++x) qn[x] = four<QUADS>(rows, at + 128 * x, x < DB - 1 ? 4 : z.D - lcol - 32 * x);
        const size_t row = row0 + min(i0 + (t & (STEP - 1)), z.Tq - 1);
        sn = reinterpret_cast<const float2*>(g.stats)[row];
        en = g.delta[row];
        if (z.mask) {
            const int i = min(i0 + ((t >> 2) & (STEP - 1)), z.Tq - 1), word = min(k0 / 32 + (t & 3), (z.Tk - 1) / 32);
            const unsigned long long* m = z.mask + b * z.mask_stride[0] + h * z.mask_stride[1] + i * z.mask_stride[2];
            mn = reinterpret_cast<const uint32_t*>(m)[word];
        }
        if (BIAS) {
            const int c = k0 + t - (STEP - 1) - i0 + z.Tq - 1;  // (outside of the bias no pair needs it)
            bn = z.bias[(size_t)h * (z.Tq + z.Tk - 1) + max(0, min(c, z.Tq + z.Tk - 2))];
        }
    };
    const auto store = [&](int i0) {
        const int t = fresh(threadIdx.x), lrow = (t >> 3) & (STEP - 1), lcol = 4 * (t & 7);
        float* to = first_half ? Qs : Ys;
#pragma unroll
        for (int x = 0; x < DB; ++x) {
            const int d = lcol + 32 * x;
            float* p = to + lrow * QS + (d & ~15) + ((d >> 2) & 3);  // values 4 s + c of sixteen at 4 c + s
#pragma unroll
            for (int c = 0; c < 4; ++c) p[4 * c] = part_of(qn[x], c);
        }
        if (t < (BIAS ? 1 : 2) * STEP) {
            const int i = i0 + (t & (STEP - 1));
            Query[t] = make_float4(t < STEP ? sn.x : 0.0f, sn.y, en, __int_as_float(i < z.Tq ? last_end(z, len, i) : 0));
        }
        if (t >= 128 && t < 256) Masks[(t >> 2) & (STEP - 1)][t & 3] = mn;
        if (BIAS && t < KEY_BLOCK + STEP - 1) Bs[t] = bias_term(bn);
    };
    const int row_of = 4 * (col & 3) + (col >> 2);    // the query of 16 that row `col` of an operand is
    const int place_in = 4 * (col & 3) + (col >> 2);  // where value `col` of 16 is in Qs and Ys

    const int first_chunk = at.part * w.a_part, last_chunk = min(w.chunks, first_chunk + w.a_part);
    bool begun = false;
    for (int chunk = first_chunk; chunk < last_chunk; ++chunk) {
        const int c0 = chunk * QUERY_CHUNK, c1 = min(c0 + QUERY_CHUNK, z.Tq);
        if (!live(z, len, block, c1)) continue;
        float* diagonals = BIAS && w.diagonals ? w.diagonals + (((size_t)bh * w.count + slot) * w.chunks + chunk) * DIAGONALS : nullptr;
        Block4 dk[2 * DB], dv[2 * DB];
#pragma unroll
        for (int n = 0; n < 2 * DB; ++n) dk[n] = dv[n] = Block4{0.0f, 0.0f, 0.0f, 0.0f};
        int i0 = c0;
        while (!live(z, len, block, i0 + STEP)) i0 += STEP;  // (the chunk's last step is live)
        __syncthreads();
        load(i0);
        store(i0);
        if (BIAS)
            for (int n = t; n < DIAGONALS; n += 512) Sums[n] = 0.0f;
        lds_barrier();
        for (; i0 < c1; i0 += STEP) {
            const bool more = i0 + STEP < c1;
            Block4 s[2], dp[2];  // register r of block n: query 16 n + 4 r + group
#pragma unroll
            for (int n = 0; n < 2; ++n) s[n] = dp[n] = Block4{0.0f, 0.0f, 0.0f, 0.0f};
            {
                const float* qs = Qs + row_of * QS + 4 * group;
                const float* ys = Ys + row_of * QS + 4 * group;
                float4 a[2], c[2];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    a[n] = *reinterpret_cast<const float4*>(qs + 16 * n * QS);
                    c[n] = *reinterpret_cast<const float4*>(ys + 16 * n * QS);
                }
#pragma unroll
                for (int u = 0; u < 2 * DB; ++u) {
                    const int ahead = 16 * (u + 1 < 2 * DB ? u + 1 : u);
                    float4 an[2], cn[2];
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        an[n] = *reinterpret_cast<const float4*>(qs + 16 * n * QS + ahead);
                        cn[n] = *reinterpret_cast<const float4*>(ys + 16 * n * QS + ahead);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            s[n] = mfma4(part_of(a[n], r), k[4 * u + r], s[n]);
                            dp[n] = mfma4(part_of(c[n], r), v[4 * u + r], dp[n]);
                        }
#pragma unroll
                    for (int n = 0; n < 2; ++n) a[n] = an[n], c[n] = cn[n];
                    fence();
                }
            }
            uint32_t keep[4];
            if (DROP) {
                // a call's four words are four keys', neighbours in a quad of lanes: each makes those of another query
                uint32_t bits = 0;
                const int r = lane & 3;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const auto x = repro_dropout::pair_words((uint32_t)(key >> 2), i0 + 16 * n + 4 * r + group, bh, seed);
#pragma unroll
                    for (int q = 0; q < 4; ++q) bits |= (uint32_t)(x.w[q] >= z.threshold) << (4 * n + q);
                }
                keep[0] = __builtin_amdgcn_update_dpp(0, bits, 0x00, 0xF, 0xF, true) >> r;
                keep[1] = __builtin_amdgcn_update_dpp(0, bits, 0x55, 0xF, 0xF, true) >> r;
                keep[2] = __builtin_amdgcn_update_dpp(0, bits, 0xAA, 0xF, 0xF, true) >> r;
                keep[3] = __builtin_amdgcn_update_dpp(0, bits, 0xFF, 0xF, 0xF, true) >> r;
            }
            const bool large = !BIAS && __any(is_large(Query[lane & (STEP - 1)].x));
            if (large) {  // the exponents are made here, and kept by what follows
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        s[n][r] = repro_attention::less(s[n][r], s[n][r] * z.factor, z.factor, Query[16 * n + 4 * r + group].x, false);
            }
            const float factor = large ? 1.0f : z.factor;
            const float4* rows = Query + (large ? STEP : 0);
            const auto differentials = [&](auto edge) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int q = 16 * n + 4 * r + group;
                        const float4 row = rows[q];
                        const float x = BIAS ? __builtin_fmaf(s[n][r], z.factor, Bs[16 * wave + col - q + STEP - 1]) - row.x
                                             : __builtin_fmaf(s[n][r], factor, -row.x);
                        float p = e2(x) * row.y, d = dp[n][r], u = p;
                        if (DROP) {
                            const bool kept = (keep[r] >> (4 * n) & 1) != 0;
                            u = kept ? p * z.keep_factor : 0.0f;
                            d = kept ? d * z.keep_factor : 0.0f;
                        }
                        d = ds_of(p, d, row.z);
                        if (decltype(edge)::value) {
                            const bool see = (int)(key < __float_as_int(row.w)) & (int)(Masks[q][wave >> 1] >> (16 * (wave & 1) + col) & 1);
                            u = see ? u : 0.0f;
                            d = see ? d : 0.0f;
                        }
                        s[n][r] = u;
                        dp[n][r] = d;
                        Ds[q * DS_STRIDE + 16 * wave + col] = d;
                    }
            };
            // whether every pair of the wavefront's is seen
            if (!z.mask && i0 + STEP <= z.Tq && k0 + 16 * wave + 16 <= last_end(z, len, i0)) differentials(std::false_type());
            else differentials(std::true_type());
            {
                const float* qs = Qs + group * QS + place_in;
                const float* ys = Ys + group * QS + place_in;
                float a[2 * DB], c[2 * DB];
#pragma unroll
                for (int x = 0; x < 2 * DB; ++x) a[x] = ys[16 * x], c[x] = qs[16 * x];
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const int ahead = 4 * (n < 7 ? n + 1 : n) * QS;
                    float an[2 * DB], cn[2 * DB];
#pragma unroll
                    for (int x = 0; x < 2 * DB; ++x) an[x] = ys[ahead + 16 * x], cn[x] = qs[ahead + 16 * x];
#pragma unroll
                    for (int x = 0; x < 2 * DB; ++x) {
                        dv[x] = mfma4(a[x], s[n / 4][n % 4], dv[x]);
                        dk[x] = mfma4(c[x], dp[n / 4][n % 4], dk[x]);
                    }
#pragma unroll
                    for (int x = 0; x < 2 * DB; ++x) a[x] = an[x], c[x] = cn[x];
                    fence();
                }
            }
            lds_barrier();
            if (more) load(i0 + STEP);  // (in flight under dQ's products)
            {
                // the wavefront's 16 queries and its blocks of 16 values: the first and, where there are as many, the one 4 on
                const int q0 = 16 * (wave & 1), x0 = wave >> 1;
                const float* ds = Ds + (q0 + col) * DS_STRIDE + group;
                const float* ks[2];
                Block4 dq[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    ks[x] = Ks + group * KS + 16 * min(x0 + 4 * x, 2 * DB - 1) + col;
                    dq[x] = Block4{0.0f, 0.0f, 0.0f, 0.0f};
                }
                float a[4], c[4][2];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    a[r] = ds[4 * r];
#pragma unroll
                    for (int x = 0; x < 2; ++x) c[r][x] = ks[x][4 * r * KS];
                }
#pragma unroll
                for (int n = 0; n < KEY_BLOCK / 16; ++n) {
                    const int ahead = 16 * (n + 1 < KEY_BLOCK / 16 ? n + 1 : n);
                    float an[4], cn[4][2];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        an[r] = ds[ahead + 4 * r];
#pragma unroll
                        for (int x = 0; x < 2; ++x) cn[r][x] = ks[x][(ahead + 4 * r) * KS];
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int x = 0; x < 2; ++x) dq[x] = mfma4(a[r], c[r][x], dq[x]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        a[r] = an[r];
#pragma unroll
                        for (int x = 0; x < 2; ++x) c[r][x] = cn[r][x];
                    }
                    fence();
                }
                const Rows rows = rows_at(w.dq + ((size_t)slot * heads * z.Tq + row0 + i0) * z.D, min(STEP, z.Tq - i0), z.D, z.D);
                const int from = fresh(lane);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int d = 16 * (x0 + 4 * x) + (from & 15);
                    const uint32_t to = x0 + 4 * x < 2 * DB && d < z.D ? ((uint32_t)(q0 + 4 * (from >> 4)) * z.D + d) * 4 : NOWHERE;
#pragma unroll
                    for (int r = 0; r < 4; ++r) put_one(rows, to + (uint32_t)(4 * r * z.D), dq[x][r]);
                }
            }
            if (BIAS && w.diagonals && t < KEY_BLOCK + STEP - 1) {
                float* sum = Sums + t - (STEP - 1) - (i0 - c0) + QUERY_CHUNK - 1;
                const float* ds = Ds + t - (STEP - 1);
                float x = *sum;
#pragma unroll
                for (int q = 0; q < STEP; ++q) x = x + ds[q * (DS_STRIDE + 1)];
                *sum = x;
            }
            if (more) store(i0 + STEP);
            lds_barrier();
        }
        const bool last = w.direct && chunk == w.chunks - 1;
        const size_t chunk_out = out_of(z, w, bh, chunk);
        const bool add = w.parts == 1 && begun;
        begun = true;
        const auto leave = [&](float* base, const Block4* sum, float scale) {
            const Rows rows = rows_at(base + chunk_out + k0 * out_stride, min(KEY_BLOCK, z.Tk - k0), out_stride, z.D);
            const int lane = fresh(threadIdx.x) & 63, group = lane >> 4;
            const uint32_t to = ((uint32_t)(16 * wave + (lane & 15)) * (uint32_t)out_stride + 4 * group) * 4;
            float4 held[2 * DB];
            if (add) {
#pragma unroll
                for (int n = 0; n < 2 * DB; ++n) held[n] = four<QUADS>(rows, to + 64 * n, z.D - 16 * n - 4 * group);
            }
#pragma unroll
            for (int n = 0; n < 2 * DB; ++n) {
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    broken = __builtin_fmaf(sum[n][r], 0.0f, broken);
                    v[r] = add ? part_of(held[n], r) + sum[n][r] : sum[n][r];
                    if (last) v[r] = v[r] * scale + 0.0f;
                }
                put_four<QUADS>(rows, to + 64 * n, z.D - 16 * n - 4 * group, v);
            }
        };
        leave(w.dk, dk, z.scale);
        leave(w.dv, dv, 1.0f);
        if (diagonals)
            for (int n = t; n < DIAGONALS; n += 512) diagonals[n] = Sums[n];
    }
    if (w.broken) {  // a NaN or infinity, which the products' zeros hand to pairs that are not seen, shows in every key's sums
        const int any = __syncthreads_or(broken != broken);
        if (t == 0) w.broken[blockIdx.x] = any;
    }
}

// Redoes the blocks whose operands hold a NaN or infinity, key by key, row by row and pair by pair.
__global__ void __launch_bounds__(256)
repair(Problem z, Gradients g, Work w) {
    if (w.broken[blockIdx.x] == 0) return;
    const uint64_t seed = z.seed_at ? *z.seed_at : z.seed;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Place at = place_of(z, w);
    const int b = at.bh / z.H, h = at.bh % z.H, heads = z.B * z.H, block = w.first + at.slot, k0 = block * KEY_BLOCK;
    const int len = keys_of(z, b), first_chunk = at.part * w.a_part, last_chunk = min(w.chunks, first_chunk + w.a_part);
    const size_t out_stride = (size_t)(w.direct ? z.KVH : 1) * z.D;
    for (int n = wave; n < KEY_BLOCK && k0 + n < z.Tk; n += 4) {
        KeyPart sum{0.0f, 0.0f, 0.0f, 0.0f};
        for (int chunk = first_chunk; chunk < last_chunk; ++chunk) {
            if (!live(z, len, block, min((chunk + 1) * QUERY_CHUNK, z.Tq))) continue;
            const KeyPart r = key_part(z, g, seed, b, h, k0 + n, chunk * QUERY_CHUNK, lane);
            if (w.parts > 1) sum = r;
            else sum.v0 = sum.v0 + r.v0, sum.v1 = sum.v1 + r.v1, sum.k0 = sum.k0 + r.k0, sum.k1 = sum.k1 + r.k1;
            if (w.parts == 1 && chunk + 1 < last_chunk) continue;
            const size_t to = out_of(z, w, at.bh, chunk) + (k0 + n) * out_stride;
            const float scale = w.direct ? z.scale : 1.0f;
            if (lane < z.D) w.dk[to + lane] = sum.k0 * scale + 0.0f, w.dv[to + lane] = sum.v0 + 0.0f;
            if (lane + 64 < z.D) w.dk[to + lane + 64] = sum.k1 * scale + 0.0f, w.dv[to + lane + 64] = sum.v1 + 0.0f;
        }
    }
    for (int chunk = first_chunk; chunk < last_chunk; ++chunk) {
        const int c0 = chunk * QUERY_CHUNK, c1 = min(c0 + QUERY_CHUNK, z.Tq);
        if (!live(z, len, block, c1)) continue;
        for (int i = c0 + wave; i < c1; i += 4) {
            const QueryPart r = query_part(z, g, seed, b, h, i, k0, last_end(z, len, i), lane);
            float* to = w.dq + ((size_t)at.slot * heads * z.Tq + (size_t)at.bh * z.Tq + i) * z.D;
            if (lane < z.D) to[lane] = r.q0;
            if (lane + 64 < z.D) to[lane + 64] = r.q1;
        }
        if (!w.diagonals) continue;
        float* diagonals = w.diagonals + (((size_t)at.bh * w.count + at.slot) * w.chunks + chunk) * DIAGONALS;
        for (int n = threadIdx.x; n < DIAGONALS; n += 256) {
            const int away = n - (QUERY_CHUNK - 1);  // key in the block less query in the chunk
            float x = 0.0f;
            for (int i = max(0, -away); i < c1 - c0 && i + away < KEY_BLOCK; ++i) {
                const int j = k0 + i + away;
                x = x + pair(z, g, seed, b, h, c0 + i, j, seen(z, b, h, c0 + i, j, last_end(z, len, c0 + i))).ds;
            }
            diagonals[n] = x;
        }
    }
}

// dq = (what it is) + the key blocks' shares, in their order; the first time 0, the last time times scale.
__global__ void __launch_bounds__(256)
sum_queries(Problem z, Work w, float* dq, int begins, int ends) {
    const long long rows = (long long)z.B * z.H * z.Tq;
    const int wide = (z.D + 63) / 64 * 64;  // a row takes whole wavefronts
    for (long long n = (long long)blockIdx.x * 256 + threadIdx.x; n < rows * wide; n += (long long)gridDim.x * 256) {
        const long long row = n / wide;
        const int d = (int)(n % wide), i = (int)(row % z.Tq), bh = (int)(row / z.Tq);
        if (d >= z.D) continue;
        float* to = dq + (((size_t)(bh / z.H) * z.Tq + i) * z.H + bh % z.H) * z.D + d;
        const int end = last_end(z, keys_of(z, bh / z.H), i);
        float s = begins ? 0.0f : *to;
        const float* p = w.dq + (size_t)row * z.D + d;
        const size_t apart = (size_t)rows * z.D;
        const int blocks = min(w.count, (end + KEY_BLOCK - 1) / KEY_BLOCK - w.first);
#pragma unroll 4
        for (int k = 0; k < blocks; ++k) s = s + p[k * apart];
        *to = ends ? s * z.scale + 0.0f : s;
    }
}

// dk and dv from the heads' (and, where they are apart, the chunks') sums.
__global__ void __launch_bounds__(256)
sum_keys(Problem z, Work w, float* dk, float* dv) {
    const int j0 = w.first * KEY_BLOCK, keys = min(z.Tk - j0, w.count * KEY_BLOCK);
    const long long count = (long long)z.B * keys * z.KVH * z.D;
    for (long long n = (long long)blockIdx.x * 256 + threadIdx.x; n < count; n += (long long)gridDim.x * 256) {
        const int d = (int)(n % z.D), kvh = (int)(n / z.D % z.KVH), j = j0 + (int)(n / z.D / z.KVH % keys);
        const int b = (int)(n / z.D / z.KVH / keys), len = keys_of(z, b);
        float sk = 0.0f, sv = 0.0f;
        for (int h = kvh * z.group; h < (kvh + 1) * z.group; ++h) {
            float ck = 0.0f, cv = 0.0f;
            for (int c = 0; c < (w.parts > 1 ? w.chunks : 1); ++c) {
                if (!live(z, len, j / KEY_BLOCK, w.parts > 1 ? (c + 1) * QUERY_CHUNK : z.Tq)) continue;
                const size_t at = ((((size_t)c * z.B + b) * z.H + h) * z.Tk + j) * z.D + d;
                ck = ck + w.dk[at];
                cv = cv + w.dv[at];
            }
            sk = sk + ck;
            sv = sv + cv;
        }
        const size_t to = (((size_t)b * z.Tk + j) * z.KVH + kvh) * z.D + d;
        dk[to] = sk * z.scale + 0.0f;
        dv[to] = sv + 0.0f;
    }
}

// The bias's gradient at each distance, over the key blocks, the batch and the chunks: a block takes 64 distances of a head, its
// wavefronts bring the terms, TERMS at a time, and one adds them up in order. A key block and item have two terms: a
// distance meets at most two chunks there.
constexpr int TERMS = 64;

__global__ void __launch_bounds__(256)
sum_diagonals(Problem z, Work w, int first_head, float* dbias, int begins, int ends) {
    __shared__ float terms[TERMS][64];
    const int columns = z.Tq + z.Tk - 1, across = (columns + 63) / 64, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = first_head + blockIdx.x / across, column = (blockIdx.x % across) * 64 + lane, away = column - (z.Tq - 1);
    const bool there = column < columns;
    float s = begins || !there || wave > 0 ? 0.0f : dbias[(size_t)h * columns + column];
    // the key blocks that one of the block's distances meets
    const int least = away - lane, k_low = max(0, least) / KEY_BLOCK, k_high = min(z.Tk - 1, z.Tq - 1 + least + 63) / KEY_BLOCK;
    const int first = max(0, k_low - w.first), last = min(w.count, k_high + 1 - w.first);
    const int count = (last - first) * z.B * 2;
    for (int at = 0; at < count; at += TERMS) {
        float v[TERMS / 4];
#pragma unroll
        for (int n = 0; n < TERMS / 4; ++n) {  // (a term that is not there is read elsewhere and left out)
            const int term = min(at + 4 * n + wave, count - 1), slot = first + term / 2 / z.B, b = term / 2 % z.B;
            const int k0 = (w.first + slot) * KEY_BLOCK, low = max(0, k0 - away), high = min(z.Tq, min(k0 + KEY_BLOCK, z.Tk) - away);
            const int chunk = low / QUERY_CHUNK + (term & 1);  // of the queries low .. high
            const bool is = at + 4 * n + wave < count && there && low < high && chunk * QUERY_CHUNK < high &&
                            live(z, keys_of(z, b), w.first + slot, (chunk + 1) * QUERY_CHUNK);
            const float x = w.diagonals[is ? ((((size_t)b * z.H + h) * w.count + slot) * w.chunks + chunk) * DIAGONALS + away - k0 +
                                                 chunk * QUERY_CHUNK + QUERY_CHUNK - 1 : 0];
            v[n] = is ? x : 0.0f;
        }
#pragma unroll
        for (int n = 0; n < TERMS / 4; ++n) terms[4 * n + wave][lane] = v[n];
        __syncthreads();
        if (wave == 0) {
#pragma unroll 16
            for (int n = 0; n < TERMS; ++n) s = s + terms[n][lane];
        }
        __syncthreads();
    }
    if (wave == 0 && there) dbias[(size_t)h * columns + column] = ends ? s + 0.0f : s;
}

// dQ's sums read what they add at the copy's rate (210 us of the 4096 x 4096 pass; making the scores again instead would
// be 2 of 7 products more, 1.3 ms).
//
// How the key blocks are taken: as many at a time as leave at most a gigabyte for dQ and half of one for the bias and make a grid of
// at most 2^22 blocks; the queries split
// over blocks, whole chunks each, where the key blocks alone leave compute units idle and the chunks' results stay below
// half a gigabyte.
struct Plan {
    Work w;
    int blocks;
    size_t kv, dq, diagonals, broken, bytes;  // workspace: offsets, and its size
};

size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }

Plan plan_of(const Problem& z, bool want_bias) {
    Plan p{};
    const size_t rows = (size_t)z.B * z.H * z.Tq, a_block = rows * z.D * sizeof(float), keys = (size_t)z.B * z.H * z.Tk * z.D * sizeof(float);
    p.blocks = (z.Tk + KEY_BLOCK - 1) / KEY_BLOCK;
    p.w.chunks = (z.Tq + QUERY_CHUNK - 1) / QUERY_CHUNK;
    const size_t diagonals = want_bias ? (size_t)z.B * z.H * p.w.chunks * DIAGONALS * sizeof(float) : 0;
    size_t at_a_time = a_block > 0 ? (1u << 30) / a_block : 1;
    if (diagonals > 0) at_a_time = std::min(at_a_time, (size_t)(1 << 29) / diagonals);
    at_a_time = std::min(at_a_time, (size_t)(MAX_BLOCKS / 2) / std::max<size_t>((size_t)z.B * z.H, 1));  // (at least four)
    p.w.count = (int)std::min(std::max<size_t>(at_a_time, 1), (size_t)p.blocks);
    const long long grid = (long long)z.B * z.H * p.w.count;
    long long parts = grid > 0 && grid < 384 ? (512 + grid - 1) / grid : 1;
    if (keys * 2 * p.w.chunks > (1u << 29)) parts = 1;
    if (parts > p.w.chunks) parts = p.w.chunks;
    p.w.a_part = parts > 0 ? (int)((p.w.chunks + parts - 1) / parts) : 0;
    p.w.parts = p.w.a_part > 0 ? (p.w.chunks + p.w.a_part - 1) / p.w.a_part : 1;
    p.w.direct = p.w.parts == 1 && z.group == 1;
    p.kv = padded(rows * sizeof(float));
    p.dq = p.kv + (p.w.direct ? 0 : padded(2 * keys * (p.w.parts > 1 ? p.w.chunks : 1)));
    p.diagonals = p.dq + padded(a_block * p.w.count);
    p.broken = p.diagonals + padded(diagonals * p.w.count);
    p.bytes = p.broken + (size_t)z.B * z.H * p.w.count * p.w.parts * sizeof(int);
    return p;
}

}  // namespace

size_t backward_workspace(const Problem& z, bool want_bias) { return plan_of(z, want_bias).bytes; }

int backward(const Problem& z, const float* dy, const float* stats, float* dq, float* dk, float* dv, float* dbias, void* workspace,
             hipStream_t stream) {
    Plan p = plan_of(z, dbias != nullptr);
    char* base = static_cast<char*>(workspace);
    const Gradients g{dy, stats, reinterpret_cast<const float*>(base)};
    Work w = p.w;
    const long long values = (long long)z.B * z.H * z.Tk * z.D * (w.parts > 1 ? w.chunks : 1);
    w.dk = w.direct ? dk : reinterpret_cast<float*>(base + p.kv);
    w.dv = w.direct ? dv : w.dk + values;
    w.dq = reinterpret_cast<float*>(base + p.dq);
    w.diagonals = dbias ? reinterpret_cast<float*>(base + p.diagonals) : nullptr;
    // a query's values must not reach keys that it does not see, nor a key's a query
    w.broken = z.causal || z.mask || z.key_lengths || z.overlap ? reinterpret_cast<int*>(base + p.broken) : nullptr;
    const int most = w.count, across = (z.Tq + z.Tk - 1 + 63) / 64, heads = (int)(MAX_BLOCKS / across);  // (of a launch of sum_diagonals)
    for (int first = 0; first < p.blocks; first += most) {
        w.first = first;
        w.count = std::min(most, p.blocks - first);
        const bool begins = first == 0, ends = first + w.count == p.blocks;
        with_size(z.D, [&](auto db) {
            with_flags(z.bias != nullptr, z.threshold != 0, z.quads != 0, [&](auto bias, auto drop, auto quads) {
                constexpr int DB = decltype(db)::value;
                constexpr bool BIAS = decltype(bias)::value, DROP = decltype(drop)::value, QUADS = decltype(quads)::value;
                const dim3 grid((unsigned)(z.B * z.H * w.count * w.parts));
                if constexpr (DB <= 2)
                    hipLaunchKernelGGL((backward_tiles<DB, BIAS, DROP, QUADS>), grid, dim3(256), 0, stream, z, g, w);
                else
                    hipLaunchKernelGGL((backward_wide<DB, BIAS, DROP, QUADS>), grid, dim3(512), 0, stream, z, g, w);
            });
        });
        if (w.broken)
            hipLaunchKernelGGL(repair, dim3((unsigned)(z.B * z.H * w.count * w.parts)), dim3(256), 0, stream, z, g, w);
        hipLaunchKernelGGL(sum_queries, dim3(grid_of((long long)z.B * z.H * z.Tq * ((z.D + 63) / 64 * 64), 256)), dim3(256), 0, stream, z,
                           w, dq, begins, ends);
        if (!w.direct)
            hipLaunchKernelGGL(sum_keys, dim3(grid_of((long long)z.B * std::min(z.Tk, w.count * KEY_BLOCK) * z.KVH * z.D, 256)), dim3(256),
                               0, stream, z, w, dk, dv);
        if (dbias)
            for (int h = 0; h < z.H; h += heads)
                hipLaunchKernelGGL(sum_diagonals, dim3((unsigned)(std::min(heads, z.H - h) * across)), dim3(256), 0, stream, z, w, h, dbias,
                                   begins, ends);
        const int rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
    }
    return hipSuccess;
}

}  // namespace attention
}  // namespace rg
