// The attention's forward pass on the matrix cores.
//
// A block takes 128 queries of a head, 32 a wavefront, and goes through the keys in tiles of 64 that its wavefronts share in LDS.
// v_mfma_f32_32x32x2_f32 adds a pair of products a step, in ascending order, each fused and rounded as fmaf is, subnormals and
// all (524288 of 524288 results the same in each of four ranges): the definition's chains. Scores are made as S^T = K Q^T, so that a
// lane holds scores of one query (column lane mod 32), and a register of the result is, as it stands, the operand of
// O^T = V^T P^T for two successive keys: row 8 g + 4 h + r of the tile's operand is taken to be key 8 g + 2 r + h, so half h
// of the wavefront holds the keys of parity h in ascending order. Nothing of the softmax passes through LDS, and a row's maximum
// takes one exchange between the halves.
//
// The float32 matrix instructions and the vector unit's take turns on a SIMD (1154 and 2141 us apart, 3247 together, where
// int8 ones overlap), so every vector instruction counts: a score costs 10.5, a kept or dropped pair 13 more (Philox's
// products). 2 x 16 heads of 4096 x 4096 x 64: 1138 us, 121 TFLOP/s of the 153 that a product of 8192^3 reaches; at
// 8 x 12 heads of 1024 the blocks are one and a half rounds: 95 to 97.
#include "rg_attention.h"

namespace rg {
namespace attention {
namespace {

typedef float Block16 __attribute__((ext_vector_type(16)));

constexpr int ROWS = 128;

__device__ __forceinline__ Block16 zero16() {
    Block16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.0f;
    return z;
}
__device__ __forceinline__ Block16 mfma(float a, float b, Block16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}
// The value of the lane 32 away.
__device__ __forceinline__ void halves(uint32_t v, uint32_t* low, uint32_t* high) {
    const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    *low = s[0];
    *high = s[1];
}

// Where the keys are split over blocks, the first part's chunks are handed on joined and the others' one by one, as m, l (-1: nothing
// was seen there) and o.
struct Parts {
    int parts, chunks, a_part, slots;  // chunks a part; slots: 1 and the chunks after the first part's
    uint32_t from;                     // blocks of earlier launches
    float2* ml;                        // [slots][B][H][Tq]
    float* o;                          // [slots][B][H][Tq][D]
    __device__ __forceinline__ int slot_of(int chunk) const { return chunk < a_part ? 0 : chunk - a_part + 1; }
    int* broken;                       // a number for each block: whether `repair` has to redo it; null where it never has to
    __device__ __forceinline__ uint32_t block() const { return from + blockIdx.x; }
};

// The block's place: head, first query, part.
struct Place {
    int bh, i0, part;
};
__device__ __forceinline__ Place place_of(const Problem& z, const Parts& s) {
    const int heads = z.B * z.H, rest = (int)(s.block() / heads);
    // under a causal mask the longest first
    return Place{(int)(s.block() % heads), ((z.Tq + ROWS - 1) / ROWS - 1 - rest / s.parts) * ROWS, rest % s.parts};
}

// DB blocks of 32 values hold a head's; QUADS as in four().
template <int DB, bool BIAS, bool DROP, bool QUADS>
__global__ void __launch_bounds__(256, 2)
forward_tiles(Problem z, Parts s, float* y, float* stats, unsigned long long* used) {
    constexpr int DP = 32 * DB, KS = DP + 4;
    constexpr bool AHEAD = DB <= 2;  // the next tile in registers while one is worked on
    __shared__ float Ks[TILE * KS], Vs[TILE * DP], Bs[BIAS ? TILE + ROWS : 1];
    const uint64_t seed = z.seed_at ? *z.seed_at : z.seed;
    if (used && blockIdx.x == 0 && threadIdx.x == 0) *used = seed;
    const int t = threadIdx.x, lane = t & 63, col = lane & 31, half = lane >> 5, wave = t >> 6;
    const Place at = place_of(z, s);
    const int bh = at.bh, b = bh / z.H, h = bh % z.H, part = at.part, i0 = at.i0;
    const int w0 = i0 + 32 * wave, i = w0 + col;
    const int len = keys_of(z, b);
    const auto end_of = [&](int last) { return z.causal ? max(0, min(len, last + z.start + 1)) : len; };
    const int block_end = end_of(min(i0 + ROWS, z.Tq) - 1);
    const int wave_end = w0 < z.Tq ? end_of(min(w0 + 32, z.Tq) - 1) : 0;
    const int row_end = i < z.Tq ? end_of(i) : 0;
    const int full = z.mask ? 0 : w0 + 32 <= z.Tq ? end_of(w0) : 0;  // keys below it are seen by the whole wavefront
    const unsigned long long* mask_row = nullptr;
    if (z.mask && i < z.Tq) mask_row = z.mask + b * z.mask_stride[0] + h * z.mask_stride[1] + i * z.mask_stride[2];

    float q[16 * DB];  // value 2 n + half of the row
    {
        const Rows rows = rows_at(query_at(z, b, h, i0), min(ROWS, z.Tq - i0), z.q_stride[1], z.D);
        const uint32_t row = (uint32_t)(32 * wave + col) * (uint32_t)z.q_stride[1] * 4;
#pragma unroll
        for (int u = 0; u < 4 * DB; ++u) {
            const float4 a = four<QUADS>(rows, row + 32 * u, z.D - 8 * u), c = four<QUADS>(rows, row + 32 * u + 16, z.D - 8 * u - 4);
            q[4 * u] = half ? a.y : a.x;
            q[4 * u + 1] = half ? a.w : a.z;
            q[4 * u + 2] = half ? c.y : c.x;
            q[4 * u + 3] = half ? c.w : c.z;
#pragma unroll
            for (int r = 0; r < 4; ++r) q[4 * u + r] = z.flip ? -q[4 * u + r] : q[4 * u + r];
        }
    }
    const int key_row = (col & 24) + 2 * (col & 3) + ((col >> 2) & 1);  // the key that row `col` of an operand is

    // a thread brings four values in each 32 of two rows of k and v
    const int lrow = t >> 3, lcol = 4 * (t & 7);
    uint32_t kat[2], vat[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        kat[n] = ((uint32_t)(lrow + 32 * n) * (uint32_t)z.k_stride[1] + lcol) * 4;
        vat[n] = ((uint32_t)(lrow + 32 * n) * (uint32_t)z.v_stride[1] + lcol) * 4;
    }
    float4 kn[2 * DB], vn[2 * DB];
    float bn = 0.0f, broken = 0.0f;
    const auto watch = [&](const Block16* sum) {
#pragma unroll
        for (int n = 0; n < 16 * DB; ++n) broken = __builtin_fmaf(sum[n / 16][n % 16], 0.0f, broken);
    };
    const float* kbase = key_at(z, b, h, 0);
    const float* vbase = value_at(z, b, h, 0);
    const auto load_keys = [&](int j0) {
        const Rows rows = rows_at(kbase + j0 * z.k_stride[1], min(TILE, len - j0), z.k_stride[1], z.D);
#pragma unroll
        for (int n = 0; n < 2 * DB; ++n) kn[n] = four<QUADS>(rows, kat[n / DB] + 128 * (n % DB), n % DB < DB - 1 ? 4 : z.D - lcol - 32 * (n % DB));
        if (BIAS) {
            const int c = j0 + t - (ROWS - 1) - i0 + z.Tq - 1;  // (outside of the bias no pair needs it)
            bn = z.bias[(size_t)h * (z.Tq + z.Tk - 1) + max(0, min(c, z.Tq + z.Tk - 2))];
        }
    };
    const auto load_values = [&](int j0) {
        const Rows rows = rows_at(vbase + j0 * z.v_stride[1], min(TILE, len - j0), z.v_stride[1], z.D);
#pragma unroll
        for (int n = 0; n < 2 * DB; ++n) vn[n] = four<QUADS>(rows, vat[n / DB] + 128 * (n % DB), n % DB < DB - 1 ? 4 : z.D - lcol - 32 * (n % DB));
    };
    const auto store_keys = [&]() {
#pragma unroll
        for (int n = 0; n < 2 * DB; ++n) {
            const int d = lcol + 32 * (n % DB);
            float* p = Ks + (lrow + n / DB * 32) * KS + (d & ~7) + (d & 4) / 2;  // values 2 r + h of eight at 4 h + r
            *reinterpret_cast<float2*>(p) = make_float2(kn[n].x, kn[n].z);
            *reinterpret_cast<float2*>(p + 4) = make_float2(kn[n].y, kn[n].w);
        }
        if (BIAS && t < TILE + ROWS - 1) Bs[t] = bias_term(bn);
    };
    const auto store_values = [&]() {
#pragma unroll
        for (int n = 0; n < 2 * DB; ++n) *reinterpret_cast<float4*>(Vs + (lrow + n / DB * 32) * DP + lcol + 32 * (n % DB)) = vn[n];
    };

    const int first_chunk = part * s.a_part, last_chunk = min(s.chunks, first_chunk + s.a_part);
    const int first_key = first_chunk * CHUNK, last_key = min(last_chunk * CHUNK, block_end);
    const size_t row_index = (size_t)bh * z.Tq + i;
    const size_t all_rows = (size_t)z.B * z.H * z.Tq;
    const auto leave = [&](int chunk, float m, float l, const Block16* sum) {
        watch(sum);
        const int slot = s.slot_of(chunk);
        const Rows rows = rows_at(s.o + (slot * all_rows + (size_t)bh * z.Tq + i0) * z.D, min(ROWS, z.Tq - i0), z.D, z.D);
        const uint32_t row = ((uint32_t)(i - i0) * z.D + 4 * half) * 4;
#pragma unroll
        for (int n = 0; n < 4 * DB; ++n) {
            const float v[4] = {sum[n / 4][4 * (n % 4)], sum[n / 4][4 * (n % 4) + 1], sum[n / 4][4 * (n % 4) + 2], sum[n / 4][4 * (n % 4) + 3]};
            put_four<QUADS>(rows, row + 32 * n, z.D - 8 * n - 4 * half, v);
        }
        if (half == 0 && i < z.Tq) s.ml[slot * all_rows + row_index] = make_float2(m, l);
    };
    float top = NONE, total = 0.0f;
    Block16 out[DB];
#pragma unroll
    for (int n = 0; n < DB; ++n) out[n] = zero16();
    if (AHEAD && first_key < last_key) {
        load_keys(first_key);
        load_values(first_key);
    }
    for (int chunk = first_chunk; chunk < last_chunk && chunk * CHUNK < block_end; ++chunk) {
        float m = NONE, l = 0.0f;
        Block16 o[DB];
#pragma unroll
        for (int n = 0; n < DB; ++n) o[n] = zero16();
        const int chunk_end = min((chunk + 1) * CHUNK, block_end);
        for (int j0 = chunk * CHUNK; j0 < chunk_end; j0 += TILE) {
            if (!AHEAD) load_keys(j0);
            lds_barrier();
            store_keys();
            if (!AHEAD) load_values(j0);
            store_values();
            lds_barrier();
            if (AHEAD && j0 + TILE < last_key) {
                load_keys(j0 + TILE);
                load_values(j0 + TILE);
            }
            if (j0 >= wave_end) continue;
            Block16 p[2] = {zero16(), zero16()};
#pragma unroll
            for (int u = 0; u < 4 * DB; ++u) {
                float4 a[2];
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    a[kb] = *reinterpret_cast<const float4*>(Ks + (32 * kb + key_row) * KS + 8 * u + 4 * half);
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
                        p[kb] = mfma(r == 0 ? a[kb].x : r == 1 ? a[kb].y : r == 2 ? a[kb].z : a[kb].w, q[4 * u + r], p[kb]);
            }
            // register 4 g + r of block kb: key j0 + 32 kb + 8 g + 2 r + half
            if (BIAS) {
                const float* bias = Bs + (ROWS - 1 - (i - i0)) + half;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        p[kb][r] = __builtin_fmaf(p[kb][r], z.factor, bias[32 * kb + 8 * (r / 4) + 2 * (r % 4)]);
            }
            // the keys of the lane's parity that its row sees, key 32 kb + n at bit n of word kb
            uint32_t see[2] = {~0u, ~0u};
            const bool edge = j0 + TILE > full;
            if (edge) {
                const unsigned long long bits = mask_row ? mask_row[j0 >> 6] : ~0ull;
                const int left = row_end - j0;
                const unsigned long long there = bits & (left >= 64 ? ~0ull : left > 0 ? (1ull << left) - 1 : 0ull);
                see[0] = (uint32_t)(there >> half);
                see[1] = (uint32_t)(there >> 32) >> half;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        p[kb][r] = (see[kb] >> (8 * (r / 4) + 2 * (r % 4)) & 1) != 0 ? p[kb][r] : -__builtin_inff();
            }
            float next = -__builtin_inff();
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 16; r += 2) next = larger(larger(next, p[kb][r]), p[kb][r + 1]);
            {
                uint32_t x, w;
                halves(__float_as_uint(next), &x, &w);
                next = larger(__uint_as_float(x), __uint_as_float(w));
            }
            next = larger(m, BIAS ? next : next * z.factor);
            const float base = base_of(next), a = rescale(m, base);
            m = next;
            l = l * a;
            if (__any(a != 1.0f)) {
#pragma unroll
                for (int n = 0; n < DB; ++n)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[n][r] = o[n][r] * a;
            }
            const bool large = !BIAS && __any(is_large(base));  // (then the exponents are made here, and kept by what follows)
            if (large) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        p[kb][r] = repro_attention::less(p[kb][r], p[kb][r] * z.factor, z.factor, base, false);
            }
            const float factor = large ? 1.0f : z.factor, shift = large ? 0.0f : base;
            const auto exponentials = [&](auto masked) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        float x = BIAS ? p[kb][r] - shift : __builtin_fmaf(p[kb][r], factor, -shift);
                        if (decltype(masked)::value) x = (see[kb] >> (8 * (r / 4) + 2 * (r % 4)) & 1) != 0 ? x : LOWEST;
                        p[kb][r] = e2(x);
                        l = l + p[kb][r];
                    }
            };
            if (edge) exponentials(std::true_type());
            else exponentials(std::false_type());
            if (DROP) {
                // the four words of a call are four keys': half 0 makes those of keys 0..3 of eight, half 1 of 4..7, and an exchange of
                // the odd words of the one with the even words of the other leaves each half those of its parity
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    const auto w = repro_dropout::pair_words((uint32_t)(j0 / 4 + 2 * g + half), i, bh, seed);
                    const auto first = __builtin_amdgcn_permlane32_swap(w.w[0], w.w[1], false, false);
                    const auto second = __builtin_amdgcn_permlane32_swap(w.w[2], w.w[3], false, false);
                    const uint32_t mine[4] = {first[0], second[0], first[1], second[1]};
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int at_r = 4 * (g % 4) + r;
                        p[g / 4][at_r] = mine[r] >= z.threshold ? p[g / 4][at_r] : 0.0f;
                    }
                }
            }
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float* v = Vs + (32 * kb + 8 * (r / 4) + 2 * (r % 4) + half) * DP + col;
#pragma unroll
                    for (int n = 0; n < DB; ++n) o[n] = mfma(v[32 * n], p[kb][r], o[n]);
                }
        }
        uint32_t x, w;
        halves(__float_as_uint(l), &x, &w);
        const float both_l = __uint_as_float(x) + __uint_as_float(w);
        if (part > 0) {
            leave(chunk, m, both_l, o);
        } else {
            const float both = larger(top, m), base = base_of(both), a = rescale(top, base), e = rescale(m, base);
            top = both;
            total = __builtin_fmaf(both_l, e, total * a);
#pragma unroll
            for (int n = 0; n < DB; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) out[n][r] = __builtin_fmaf(o[n][r], e, out[n][r] * a);
        }
    }
    if (part > 0 && i < z.Tq && half == 0)
        for (int chunk = max(first_chunk, (block_end + CHUNK - 1) / CHUNK); chunk < last_chunk; ++chunk)
            s.ml[s.slot_of(chunk) * all_rows + row_index] = make_float2(NONE, -1.0f);
    if (part == 0 && s.parts > 1) leave(0, top, total, out);
    if (s.parts == 1) watch(out);
    if (s.broken) {  // a NaN or infinity in v, which the products' zeros hand to rows that do not see it, shows in every row
        const int any = __syncthreads_or(broken != broken);
        if (t == 0) s.broken[s.block()] = any;
    }
    if (s.parts == 1) {
        const float inverse = reciprocal(total), f = DROP ? inverse * z.keep_factor : inverse;
        if (i < z.Tq) {
            const Rows rows = rows_at(y + (((size_t)b * z.Tq + i0) * z.H + h) * z.D, min(ROWS, z.Tq - i0), (long long)z.H * z.D, z.D);
            const uint32_t row = ((uint32_t)(i - i0) * (uint32_t)(z.H * z.D) + 4 * half) * 4;
#pragma unroll
            for (int n = 0; n < DB; ++n)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = out[n][4 * g + r] * f + 0.0f;
                    put_four<QUADS>(rows, row + 128 * n + 32 * g, z.D - 32 * n - 8 * g - 4 * half, v);
                }
            if (stats && half == 0) {
                stats[2 * row_index] = base_of(top);
                stats[2 * row_index + 1] = inverse;
            }
        }
    }
}

// Redoes the blocks whose values hold a NaN or infinity, row by row and pair by pair.
__global__ void __launch_bounds__(256)
repair(Problem z, Parts s, float* y, float* stats) {
    if (s.broken[s.block()] == 0) return;
    const uint64_t seed = z.seed_at ? *z.seed_at : z.seed;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Place at = place_of(z, s);
    const int b = at.bh / z.H, h = at.bh % z.H, len = keys_of(z, b);
    const int block_end = z.causal ? max(0, min(len, min(at.i0 + ROWS, z.Tq) + z.start)) : len;
    const int first_chunk = at.part * s.a_part, last_chunk = min(s.chunks, first_chunk + s.a_part);
    for (int row = at.i0 + wave; row < at.i0 + ROWS && row < z.Tq; row += 4) {
        const int end = key_end(z, b, row);
        const size_t n = (size_t)at.bh * z.Tq + row;
        Joined all;
        for (int chunk = first_chunk; chunk < last_chunk && chunk * CHUNK < block_end; ++chunk) {
            const RowChunk r = row_chunk(z, seed, b, h, row, chunk * CHUNK, end, lane);
            if (at.part > 0) {
                const size_t to = s.slot_of(chunk) * (size_t)z.B * z.H * z.Tq + n;
                if (lane < z.D) s.o[to * z.D + lane] = r.o0;
                if (lane + 64 < z.D) s.o[to * z.D + lane + 64] = r.o1;
                if (lane == 0) s.ml[to] = make_float2(r.m, r.even + r.odd);
            } else {
                all.join(r);
            }
        }
        if (s.parts == 1) finish_row(z, all, b, h, row, lane, y, stats);
        else if (at.part == 0) {
            if (lane < z.D) s.o[n * z.D + lane] = all.o0;
            if (lane + 64 < z.D) s.o[n * z.D + lane + 64] = all.o1;
            if (lane == 0) s.ml[n] = make_float2(all.top, all.total);
        }
    }
}

// Few queries: a block takes a chunk of keys for up to FEW of the rows that share a head of keys, a thread a key for the
// scores, then a wavefront a row and a lane a value. Bound by HBM: the keys are read into LDS as the values are on their way, and the
// values take their place there. One query of 2048 to 4096 keys for 16 items of 12 heads of 64: 73 us and 5.1 to join the
// chunks, 4.9 TB/s of the 5.25 of a copy; heads of 128, whose keys leave room for one block a compute unit: 3.4.
constexpr int FEW = 8;

template <int DB, bool QUADS>
__global__ void __launch_bounds__(256, DB <= 2 ? 2 : 1)
few_rows(Problem z, Parts s, float* y, float* stats, unsigned long long* used) {
    constexpr int DP = 32 * DB, STRIDE = DP + 4;
    __shared__ float KV[CHUNK * STRIDE], Qs[FEW][DP], Tops[FEW][4], Ls[FEW][2];
    __shared__ __attribute__((aligned(16))) float P[FEW][CHUNK];
    __shared__ unsigned long long See[FEW][4];
    const uint64_t seed = z.seed_at ? *z.seed_at : z.seed;
    if (used && blockIdx.x == 0 && threadIdx.x == 0) *used = seed;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int heads = z.B * z.KVH, shares = (z.group * z.Tq + FEW - 1) / FEW, chunk = (int)(s.block() / heads / shares);
    const int r0 = (int)(s.block() / heads % shares) * FEW;
    const int b = (int)(s.block() % heads) / z.KVH, kvh = (int)(s.block() % heads) % z.KVH, h0 = kvh * z.group;
    const int rows = min(FEW, z.group * z.Tq - r0), first = chunk * CHUNK;
    const int len = key_end(z, b, z.Tq - 1);  // what no row sees is not read
    const auto row_of = [&](int r) { return ((size_t)b * z.H + h0 + (r0 + r) / z.Tq) * z.Tq + (r0 + r) % z.Tq; };
    if (s.chunks > 1 && first >= len) {
        if (t < rows) s.ml[(size_t)chunk * z.B * z.H * z.Tq + row_of(t)] = make_float2(NONE, -1.0f);
        return;
    }
    const int lrow = t >> 3, lcol = 4 * (t & 7);
    const auto load = [&](const float* base, long long stride, float4* to) {
        const uint32_t at = ((uint32_t)lrow * (uint32_t)stride + lcol) * 4;
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // (128 rows are what the offsets reach)
            const Rows from = rows_at(base + (long long)(first + 128 * half) * stride, min(128, len - first - 128 * half), stride, z.D);
#pragma unroll
            for (int n = 0; n < 4 * DB; ++n)
                to[4 * DB * half + n] = four<QUADS>(from, at + 128 * (n % DB) + n / DB * 128 * (uint32_t)stride, z.D - lcol - 32 * (n % DB));
        }
    };
    const auto store = [&](const float4* from) {
#pragma unroll
        for (int n = 0; n < 8 * DB; ++n) *reinterpret_cast<float4*>(KV + (lrow + n / DB * 32) * STRIDE + lcol + 32 * (n % DB)) = from[n];
    };
    float4 held[8 * DB], next[8 * DB];
    load(key_at(z, b, h0, 0), z.k_stride[1], held);
    load(value_at(z, b, h0, 0), z.v_stride[1], next);
    for (int n = t; n < rows * DP; n += 256) {
        const int r = n / DP, d = n % DP;
        const float x = d < z.D ? query_at(z, b, h0 + (r0 + r) / z.Tq, (r0 + r) % z.Tq)[d] : 0.0f;
        Qs[r][d] = z.flip ? -x : x;
    }
    store(held);
    __syncthreads();

    const int j = first + t;
    float sum[FEW];
#pragma unroll
    for (int r = 0; r < FEW; ++r) sum[r] = 0.0f;
    for (int d = 0; d < DP; d += 4) {
        const float4 k = *reinterpret_cast<const float4*>(KV + t * STRIDE + d);
#pragma unroll
        for (int r = 0; r < FEW; ++r) {
            if (r >= rows) break;
            const float4 q = *reinterpret_cast<const float4*>(&Qs[r][d]);
            sum[r] = __builtin_fmaf(q.x, k.x, sum[r]);
            sum[r] = __builtin_fmaf(q.y, k.y, sum[r]);
            sum[r] = __builtin_fmaf(q.z, k.z, sum[r]);
            sum[r] = __builtin_fmaf(q.w, k.w, sum[r]);
        }
    }
    float term[FEW];
    bool see[FEW];
#pragma unroll
    for (int r = 0; r < FEW; ++r) {
        if (r >= rows) break;
        const int i = (r0 + r) % z.Tq, h = h0 + (r0 + r) / z.Tq;
        see[r] = seen(z, b, h, i, j, key_end(z, b, i));
        term[r] = see[r] ? z.bias ? __builtin_fmaf(sum[r], z.factor, bias_term(z.bias[(size_t)h * (z.Tq + z.Tk - 1) + j - i + z.Tq - 1]))
                                  : sum[r] * z.factor : NONE;
        const float top = wave_max(term[r]);
        const unsigned long long which = __ballot(see[r]);
        if (lane == 0) {
            Tops[r][wave] = top;
            See[r][wave] = which;
        }
    }
    __syncthreads();
    store(next);
#pragma unroll
    for (int r = 0; r < FEW; ++r) {
        if (r >= rows) break;
        float m = NONE;
        for (int w = 0; w <= wave; ++w) m = larger(m, Tops[r][w]);
        const float base = base_of(m);
        const float p = see[r] ? e2(less(z, Score{sum[r], term[r]}, base)) : 0.0f;
        P[r][t] = p;
    }
    __syncthreads();

    // the tiles' factors: what was there is multiplied by before a tile's terms come in
    const auto factors = [&](int r, float* a) {
        float m = NONE;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float up = larger(m, Tops[r][w]);
            a[w] = rescale(m, base_of(up));
            m = up;
        }
        return m;
    };
    const int tiles = min(4, (len - first + 63) / 64);  // past the keys nothing changes
    // l by the last wavefront where it has no row, or where o leaves pairs out; else it comes along with o
    const bool apart = rows < 4 || z.threshold != 0;
    if (apart && t >= 192 && t < 192 + 2 * rows) {
        const int r = (t - 192) >> 1, parity = t & 1;
        float a[4], l = 0.0f;
        factors(r, a);
        for (int w = 0; w < tiles; ++w) {
            l = l * a[w];
#pragma unroll 16
            for (int n = 0; n < 32; ++n) l = l + P[r][64 * w + 2 * n + parity];
        }
        Ls[r][parity] = l;
    }
    if (z.threshold != 0) {
        __syncthreads();
        for (int r = 0; r < rows; ++r) P[r][t] = kept(z, seed, b, h0 + (r0 + r) / z.Tq, (r0 + r) % z.Tq, j) ? P[r][t] : 0.0f;
        __syncthreads();
    }
    const bool some = z.causal || z.mask || z.overlap;
    RowChunk mine[2];  // of rows wave and wave + 4
    float a[2][4];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        mine[x].m = factors(wave + 4 * x < rows ? wave + 4 * x : 0, a[x]);
        mine[x].o0 = mine[x].o1 = mine[x].even = mine[x].odd = 0.0f;
    }
    const auto products = [&](auto both, auto alone) {
        constexpr int N = decltype(both)::value ? 2 : 1;
        for (int w = 0; w < tiles; ++w) {
            unsigned long long which = ~0ull;
#pragma unroll
            for (int x = 0; x < N; ++x) {
                mine[x].o0 = mine[x].o0 * a[x][w];
                mine[x].o1 = mine[x].o1 * a[x][w];
                mine[x].even = mine[x].even * a[x][w];
                mine[x].odd = mine[x].odd * a[x][w];
                if (some) which &= See[wave + 4 * x][w];
            }
            const float* v = KV + 64 * w * STRIDE + lane;
            if (which == ~0ull) {
#pragma unroll 4
                for (int n = 0; n < 64; n += 4) {
                    float4 p[N];
#pragma unroll
                    for (int x = 0; x < N; ++x) p[x] = *reinterpret_cast<const float4*>(&P[wave + 4 * x][64 * w + n]);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float v0 = v[(n + q) * STRIDE], v1 = DB > 2 ? v[(n + q) * STRIDE + 64] : 0.0f;
#pragma unroll
                        for (int x = 0; x < N; ++x) {
                            const float u = q == 0 ? p[x].x : q == 1 ? p[x].y : q == 2 ? p[x].z : p[x].w;
                            mine[x].o0 = __builtin_fmaf(u, v0, mine[x].o0);
                            if (DB > 2) mine[x].o1 = __builtin_fmaf(u, v1, mine[x].o1);
                            if (!decltype(alone)::value) {
                                float& l = q % 2 == 0 ? mine[x].even : mine[x].odd;
                                l = l + u;
                            }
                        }
                    }
                }
            } else {
                for (int x = 0; x < N; ++x)
                    for (int n = 0; n < 64; ++n) {  // what an unseen key holds stays out
                        if ((See[wave + 4 * x][w] >> n & 1) == 0) continue;
                        const float u = P[wave + 4 * x][64 * w + n];
                        mine[x].o0 = __builtin_fmaf(u, v[n * STRIDE], mine[x].o0);
                        if (DB > 2) mine[x].o1 = __builtin_fmaf(u, v[n * STRIDE + 64], mine[x].o1);
                        if (!decltype(alone)::value) {
                            float& l = n % 2 == 0 ? mine[x].even : mine[x].odd;
                            l = l + u;
                        }
                    }
            }
        }
    };
    if (wave + 4 < rows && apart) products(std::true_type(), std::true_type());
    else if (wave + 4 < rows) products(std::true_type(), std::false_type());
    else if (wave < rows && apart) products(std::false_type(), std::true_type());
    else if (wave < rows) products(std::false_type(), std::false_type());
    __syncthreads();
#pragma unroll
    for (int x = 0; x < FEW / 4; ++x) {
        const int r = wave + 4 * x;
        if (r >= rows) break;
        RowChunk& c = mine[x];
        if (apart) {
            c.even = Ls[r][0];
            c.odd = Ls[r][1];
        }
        if (s.chunks > 1) {
            const size_t at = (size_t)chunk * z.B * z.H * z.Tq + row_of(r);
            if (lane < z.D) s.o[at * z.D + lane] = c.o0;
            if (lane + 64 < z.D) s.o[at * z.D + lane + 64] = c.o1;
            if (lane == 0) s.ml[at] = make_float2(c.m, c.even + c.odd);
        } else {
            Joined all;
            all.join(c);
            finish_row(z, all, b, h0 + (r0 + r) / z.Tq, (r0 + r) % z.Tq, lane, y, stats);
        }
    }
}

// Joins the chunks of a row in their order: a wavefront takes a row, first a lane a chunk (the maxima before it and the
// two factors), then a lane a value (WIDE: two), with the next chunks' on the way.
template <bool WIDE>
__global__ void __launch_bounds__(256)
join_chunks(Problem z, Parts s, float* y, float* stats) {
    const int lane = threadIdx.x & 63;
    const long long rows = (long long)z.B * z.H * z.Tq;
    for (long long n = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); n < rows; n += (long long)gridDim.x * 4) {
        const int i = (int)(n % z.Tq), bh = (int)(n / z.Tq);
        Joined all;
        for (int first = 0; first < s.slots; first += 64) {
            const int c = first + lane;
            const float2 ml = c < s.slots ? s.ml[c * rows + n] : make_float2(NONE, -1.0f);
            const bool there = ml.y != -1.0f;
            float run = ml.x;  // the largest of the chunks up to this one
#pragma unroll
            for (int step = 1; step < 64; step *= 2) {
                const float before = __shfl_up(run, step, 64);
                if (lane >= step) run = larger(before, run);
            }
            run = larger(all.top, run);
            float before = __shfl_up(run, 1, 64);
            if (lane == 0) before = all.top;
            const float base = base_of(run);
            const float a = there ? rescale(before, base) : 1.0f, e = there ? rescale(ml.x, base) : 0.0f;
            const unsigned long long which = __ballot(there);
            all.top = __shfl(run, 63, 64);
            const float* o = s.o + (first * rows + n) * z.D;
            const int count = min(64, s.slots - first);
            const int d0 = min(lane, z.D - 1), d1 = min(lane + 64, z.D - 1);
            constexpr int AHEAD = WIDE ? 16 : 32;
            for (int k0 = 0; k0 < count; k0 += AHEAD) {
                float o0[AHEAD], o1[AHEAD];
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    if (k % 8 == 0 && k0 + k >= count) break;
                    const float* p = o + min(k0 + k, count - 1) * rows * z.D;
                    o0[k] = p[d0];
                    o1[k] = WIDE ? p[d1] : 0.0f;
                }
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {  // (a chunk that was not written has factors 1 and 0)
                    if (k % 8 == 0 && k0 + k >= count) break;
                    const float ak = __shfl(a, k0 + k, 64), ek = __shfl(e, k0 + k, 64), lk = __shfl(ml.y, k0 + k, 64);
                    const bool is = (which >> (k0 + k) & 1) != 0;
                    all.total = __builtin_fmaf(is ? lk : 0.0f, ek, all.total * ak);
                    all.o0 = __builtin_fmaf(is ? o0[k] : 0.0f, ek, all.o0 * ak);
                    if (WIDE) all.o1 = __builtin_fmaf(is ? o1[k] : 0.0f, ek, all.o1 * ak);
                }
            }
        }
        finish_row(z, all, bh / z.H, bh % z.H, i, lane, y, stats);
    }
}

// The same where there are few chunks (at most SLOTS): a thread takes four values of a row and works out the factors itself.
constexpr int SLOTS = 8;

template <bool QUADS>
__global__ void __launch_bounds__(256)
join_few(Problem z, Parts s, float* y, float* stats) {
    const int quads = (z.D + 3) / 4;
    const long long rows = (long long)z.B * z.H * z.Tq;
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < rows * quads; at += (long long)gridDim.x * 256) {
        const long long n = at / quads;
        const int d = 4 * (int)(at % quads), i = (int)(n % z.Tq), bh = (int)(n / z.Tq);
        float2 ml[SLOTS];
        float v[SLOTS][4];
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) {
            const long long from = min(k, s.slots - 1) * rows + n;
            ml[k] = s.ml[from];
            const float* p = s.o + from * z.D + d;
            if (QUADS) {
                const float4 x = *reinterpret_cast<const float4*>(p);
                v[k][0] = x.x, v[k][1] = x.y, v[k][2] = x.z, v[k][3] = x.w;
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) v[k][r] = p[d + r < z.D ? r : 0];
            }
        }
        float top = NONE, total = 0.0f, o[4] = {};
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) {
            if (k >= s.slots || ml[k].y == -1.0f) continue;
            const float both = larger(top, ml[k].x), base = base_of(both), a = rescale(top, base), e = rescale(ml[k].x, base);
            top = both;
            total = __builtin_fmaf(ml[k].y, e, total * a);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = __builtin_fmaf(v[k][r], e, o[r] * a);
        }
        const float inverse = reciprocal(total), f = z.threshold == 0 ? inverse : inverse * z.keep_factor;
        float* out = y + (((size_t)(bh / z.H) * z.Tq + i) * z.H + bh % z.H) * z.D + d;
        if (QUADS) {
            *reinterpret_cast<float4*>(out) = make_float4(o[0] * f + 0.0f, o[1] * f + 0.0f, o[2] * f + 0.0f, o[3] * f + 0.0f);
        } else {
            for (int r = 0; r < 4; ++r)
                if (d + r < z.D) out[r] = o[r] * f + 0.0f;
        }
        if (stats && d == 0) {
            stats[2 * n] = base_of(top);
            stats[2 * n + 1] = inverse;
        }
    }
}

// The keys are split over blocks where the queries alone leave compute units idle: up to 384 blocks, three quarters of the two a
// compute unit that fit, into as many parts as bring the grid to those, whole chunks each, as long as the chunks' results take at most a quarter of a
// gigabyte. In parts and in one, us: 64 blocks (1024 x 1024 x 64) 34, 84; 384 blocks 132, 149; 448 blocks 167, 150; 512 x 1500 x 64: 288
// blocks 186, 221; 384 blocks 190, 222; 432 blocks 241, 224.
// Up to FEW rows of a head of keys go to the kernel above, and up to 128 of at most 4 queries. There and here, us, 16 items over 12 heads of 2048 keys
// of 64: 8 rows of one head 76, 107; 9 rows 99, 107; 12 rows 115, 108; 4 queries of 4 heads 135, 371, of 8 heads 260, 571. It would still win at 5 to 8
// queries of shared heads (8 of 4 heads 258, 372; 12: 382, 372) and past 128 rows (4 items of 144: 287, 2590), with its chunks' results without a bound.
bool few(const Problem& z) { return z.Tk > 0 && ((long long)z.group * z.Tq <= FEW || (z.Tq <= 4 && (long long)z.group * z.Tq <= 128)); }
Parts parts_of(const Problem& z) {
    Parts s;
    s.chunks = (z.Tk + CHUNK - 1) / CHUNK;
    s.ml = nullptr;
    s.o = nullptr;
    s.broken = nullptr;
    s.from = 0;
    if (few(z)) {
        s.parts = s.slots = s.chunks;
        s.a_part = 1;
        return s;
    }
    const long long blocks = (long long)z.B * z.H * ((z.Tq + ROWS - 1) / ROWS);
    long long parts = blocks > 0 ? (512 + blocks - 1) / blocks : 1;
    if (blocks > 384 || (long long)z.B * z.H * z.Tq * s.chunks * (z.D + 2) > (1ll << 26)) parts = 1;
    if (parts > s.chunks) parts = s.chunks;
    s.a_part = parts > 0 ? (int)((s.chunks + parts - 1) / parts) : 0;
    s.parts = s.a_part > 0 ? (s.chunks + s.a_part - 1) / s.a_part : 1;
    if (s.parts == 1) s.a_part = s.chunks;
    s.slots = 1 + s.chunks - s.a_part;
    return s;
}
long long blocks_of(const Problem& z, const Parts& s) {
    return few(z) ? (long long)z.B * z.KVH * ((z.group * z.Tq + FEW - 1) / FEW) * s.chunks
                  : (long long)z.B * z.H * ((z.Tq + ROWS - 1) / ROWS) * s.parts;
}
// What a key holds must not reach a row that does not see it: under a causal mask or one of pairs, or where rows past the last are not 0.
// (Few rows leave out each pair by itself.)
bool watched(const Problem& z, bool masked) { return !few(z) && (z.causal || masked || z.overlap); }
size_t sums_offset(const Problem& z, const Parts& s) { return ((size_t)z.B * z.H * z.Tq * s.slots * sizeof(float2) + 15) / 16 * 16; }
size_t parts_bytes(const Problem& z, const Parts& s) {
    return s.parts > 1 ? (sums_offset(z, s) + (size_t)z.B * z.H * z.Tq * s.slots * z.D * sizeof(float) + 15) / 16 * 16 : 0;
}

}  // namespace

size_t forward_workspace(const Problem& z, bool masked) {
    const Parts s = parts_of(z);
    return parts_bytes(z, s) + (watched(z, masked) ? blocks_of(z, s) * sizeof(int) : 0);
}

int forward(const Problem& z, float* y, float* stats, unsigned long long* used, void* workspace, hipStream_t stream) {
    Parts s = parts_of(z);
    const long long rows = (long long)z.B * z.H * z.Tq, blocks = blocks_of(z, s);
    if (blocks > UINT32_MAX) return hipErrorInvalidValue;
    if (s.parts > 1) {
        s.ml = static_cast<float2*>(workspace);
        s.o = reinterpret_cast<float*>(static_cast<char*>(workspace) + sums_offset(z, s));
    }
    if (watched(z, z.mask != nullptr)) s.broken = reinterpret_cast<int*>(static_cast<char*>(workspace) + parts_bytes(z, s));
    int rc = hipSuccess;
    for (long long from = 0; from < blocks && rc == hipSuccess; from += MAX_BLOCKS) {
        s.from = (uint32_t)from;
        const dim3 grid((unsigned)std::min(blocks - from, MAX_BLOCKS));
        with_size(z.D, [&](auto db) {
            if (few(z)) {
                auto kernel = z.quads ? few_rows<decltype(db)::value, true> : few_rows<decltype(db)::value, false>;
                hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, z, s, y, stats, used);
                return;
            }
            with_flags(z.bias != nullptr, z.threshold != 0, z.quads != 0, [&](auto bias, auto drop, auto quads) {
                constexpr int DB = decltype(db)::value;
                constexpr bool BIAS = decltype(bias)::value, DROP = decltype(drop)::value, QUADS = decltype(quads)::value;
                hipLaunchKernelGGL((forward_tiles<DB, BIAS, DROP, QUADS>), grid, dim3(256), 0, stream, z, s, y, stats, used);
            });
        });
        if (s.broken) hipLaunchKernelGGL(repair, grid, dim3(256), 0, stream, z, s, y, stats);
        rc = hipGetLastError();
    }
    if (rc == hipSuccess && s.parts > 1) {
        if (s.slots <= SLOTS)
            hipLaunchKernelGGL(z.quads ? join_few<true> : join_few<false>, dim3(grid_of(rows * ((z.D + 3) / 4), 256)), dim3(256), 0, stream, z,
                               s, y, stats);
        else
            hipLaunchKernelGGL(z.D > 64 ? join_chunks<true> : join_chunks<false>, dim3(grid_of(rows, 4)), dim3(256), 0, stream, z, s, y,
                               stats);
        rc = hipGetLastError();
    }
    return rc;
}

}  // namespace attention
}  // namespace rg
