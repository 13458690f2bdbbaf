#pragma once
// What the attention's kernels share: its operands, which pairs are seen, and a wavefront's work on one row or key in the
// order of repro_attention_math.h. Internal.
#include "rg_internal.h"
#include "repro_attention.h"
#include "repro_attention_math.h"
#include "repro_dropout_math.h"

#include <algorithm>
#include <type_traits>

namespace rg {
namespace attention {

using repro_attention::base_of;
using repro_attention::bias_term;
using repro_attention::CHUNK;
using repro_attention::ds_of;
using repro_attention::e2;
using repro_attention::KEY_BLOCK;
using repro_attention::is_large;
using repro_attention::larger;
using repro_attention::LOWEST;
using repro_attention::NONE;
using repro_attention::QUERY_CHUNK;
using repro_attention::reciprocal;
using repro_attention::rescale;
using repro_attention::TILE;

struct Problem {
    const float *q, *k, *v;
    const long long* key_lengths;
    const unsigned long long* mask;
    const float* bias;
    const unsigned long long* seed_at;
    unsigned long long seed;
    int B, Tq, Tk, H, KVH, D, group, causal, start;
    int quads;  // whether all operands' rows can be taken 16 bytes at a time
    int overlap;                       // whether rows of an operand overlap: what lies past the last of them is then not read as 0
    int flip;                          // a negative scale: scores are multiplied by -1, and factor is positive
    float factor, scale, keep_factor;
    uint32_t threshold;
    long long q_stride[3], k_stride[3], v_stride[3], mask_stride[3];
};
struct Gradients {
    const float *dy, *stats, *delta;
};

// Rows of 64-bit strides: a cache may be longer than 2^32 values.
__device__ __forceinline__ const float* query_at(const Problem& z, int b, int h, int i) {
    return z.q + b * z.q_stride[0] + i * z.q_stride[1] + h * z.q_stride[2];
}
__device__ __forceinline__ const float* key_at(const Problem& z, int b, int h, int j) {
    return z.k + b * z.k_stride[0] + j * z.k_stride[1] + h / z.group * z.k_stride[2];
}
__device__ __forceinline__ const float* value_at(const Problem& z, int b, int h, int j) {
    return z.v + b * z.v_stride[0] + j * z.v_stride[1] + h / z.group * z.v_stride[2];
}
// The batch item's keys.
__device__ __forceinline__ int keys_of(const Problem& z, int b) {
    if (!z.key_lengths) return z.Tk;
    const long long n = z.key_lengths[b];
    return n < 0 ? 0 : n < z.Tk ? (int)n : z.Tk;
}
// The keys from which on query i sees none, the mask aside.
__device__ __forceinline__ int key_end(const Problem& z, int b, int i) {
    const int n = keys_of(z, b);
    return z.causal ? max(0, min(n, i + z.start + 1)) : n;
}
__device__ __forceinline__ bool seen(const Problem& z, int b, int h, int i, int j, int end) {
    if (j >= end) return false;
    if (!z.mask) return true;
    return (z.mask[b * z.mask_stride[0] + h * z.mask_stride[1] + i * z.mask_stride[2] + (j >> 6)] >> (j & 63) & 1) != 0;
}
__device__ __forceinline__ float dot(const float* a, const float* b, int D) {
    float s = 0.0f;
    for (int d = 0; d < D; ++d) s = __builtin_fmaf(a[d], b[d], s);
    return s;
}
// t, and its difference to a maximum.
struct Score {
    float s, t;
};
__device__ __forceinline__ Score score(const Problem& z, int b, int h, int i, int j) {
    float s = dot(query_at(z, b, h, i), key_at(z, b, h, j), z.D);
    s = z.flip ? -s : s;
    if (!z.bias) return Score{s, s * z.factor};
    return Score{s, __builtin_fmaf(s, z.factor, bias_term(z.bias[(size_t)h * (z.Tq + z.Tk - 1) + j - i + z.Tq - 1]))};
}
__device__ __forceinline__ float less(const Problem& z, const Score& a, float m) {
    return repro_attention::less(a.s, a.t, z.factor, m, z.bias != nullptr);
}
__device__ __forceinline__ bool kept(const Problem& z, uint64_t seed, int b, int h, int i, int j) {
    if (z.threshold == 0) return true;
    return repro_dropout::pair_words(j >> 2, i, b * z.H + h, seed).w[j & 3] >= z.threshold;
}

// A row's share of a chunk of keys; lane d holds o_d and o_{d + 64}.
struct RowChunk {
    float m, even, odd, o0, o1;
};
__device__ __forceinline__ RowChunk row_chunk(const Problem& z, uint64_t seed, int b, int h, int i, int first, int end, int lane) {
    RowChunk r{NONE, 0.0f, 0.0f, 0.0f, 0.0f};
    for (int j0 = first; j0 < first + CHUNK && j0 < end; j0 += TILE) {
        const int j = j0 + lane;
        const bool see = seen(z, b, h, i, j, end);
        const Score t = see ? score(z, b, h, i, j) : Score{NONE, NONE};
        const float next = larger(r.m, wave_max(t.t));
        const float a = rescale(r.m, base_of(next));
        r.m = next;
        r.even = r.even * a, r.odd = r.odd * a, r.o0 = r.o0 * a, r.o1 = r.o1 * a;
        const float p = see ? e2(less(z, t, base_of(next))) : 0.0f;
        const float u = see && kept(z, seed, b, h, i, j) ? p : 0.0f;
        const unsigned long long which = __ballot(see);
        for (int n = 0; n < TILE; n += 2) {
            r.even = r.even + __shfl(p, n, 64);
            r.odd = r.odd + __shfl(p, n + 1, 64);
        }
        for (int n = 0; n < TILE; ++n) {
            const float w = __shfl(u, n, 64);
            if ((which >> n & 1) == 0) continue;
            const float* v = value_at(z, b, h, j0 + n);
            if (lane < z.D) r.o0 = __builtin_fmaf(w, v[lane], r.o0);
            if (lane + 64 < z.D) r.o1 = __builtin_fmaf(w, v[lane + 64], r.o1);
        }
    }
    return r;
}
struct Joined {
    float top = NONE, total = 0.0f, o0 = 0.0f, o1 = 0.0f;
    __device__ __forceinline__ void join(const RowChunk& r) {
        const float both = larger(top, r.m), a = rescale(top, base_of(both)), e = rescale(r.m, base_of(both));
        top = both;
        total = __builtin_fmaf(r.even + r.odd, e, total * a);
        o0 = __builtin_fmaf(r.o0, e, o0 * a);
        o1 = __builtin_fmaf(r.o1, e, o1 * a);
    }
};

__device__ __forceinline__ void finish_row(const Problem& z, const Joined& all, int b, int h, int i, int lane, float* y, float* stats) {
    const float inverse = reciprocal(all.total), f = z.threshold == 0 ? inverse : inverse * z.keep_factor;
    float* out = y + (((size_t)b * z.Tq + i) * z.H + h) * z.D;
    if (lane < z.D) out[lane] = all.o0 * f + 0.0f;
    if (lane + 64 < z.D) out[lane + 64] = all.o1 * f + 0.0f;
    if (stats && lane == 0) {
        const size_t n = ((size_t)b * z.H + h) * z.Tq + i;
        stats[2 * n] = base_of(all.top);
        stats[2 * n + 1] = inverse;
    }
}

// u = p kept factor and ds of one pair, 0 where it is not seen.
struct Pair {
    float u, ds;
};
__device__ __forceinline__ Pair pair(const Problem& z, const Gradients& g, uint64_t seed, int b, int h, int i, int j, bool see) {
    if (!see) return Pair{0.0f, 0.0f};
    const size_t n = ((size_t)b * z.H + h) * z.Tq + i;
    const float p = e2(less(z, score(z, b, h, i, j), g.stats[2 * n])) * g.stats[2 * n + 1];
    float u = p, dp = dot(g.dy + (((size_t)b * z.Tq + i) * z.H + h) * z.D, value_at(z, b, h, j), z.D);
    if (z.threshold != 0) {
        const bool keep = kept(z, seed, b, h, i, j);
        u = keep ? p * z.keep_factor : 0.0f;
        dp = keep ? dp * z.keep_factor : 0.0f;
    }
    return Pair{u, ds_of(p, dp, g.delta[n])};
}

// A key's share of a chunk of queries under a head; lane d holds dv_d, dv_{d + 64}, dk_d and dk_{d + 64}.
struct KeyPart {
    float v0, v1, k0, k1;
};
__device__ __forceinline__ KeyPart key_part(const Problem& z, const Gradients& g, uint64_t seed, int b, int h, int j, int first,
                                            int lane) {
    KeyPart r{0.0f, 0.0f, 0.0f, 0.0f};
    for (int i0 = first; i0 < first + QUERY_CHUNK && i0 < z.Tq; i0 += 64) {
        const int i = i0 + lane;
        const bool see = i < z.Tq && seen(z, b, h, i, j, key_end(z, b, i));
        const Pair w = pair(z, g, seed, b, h, i, j, see);
        const unsigned long long which = __ballot(see);
        for (int n = 0; n < 64; ++n) {
            const float u = __shfl(w.u, n, 64), ds = __shfl(w.ds, n, 64);
            if ((which >> n & 1) == 0) continue;
            const float* a = g.dy + (((size_t)b * z.Tq + i0 + n) * z.H + h) * z.D;
            const float* x = query_at(z, b, h, i0 + n);
            if (lane < z.D) {
                r.v0 = __builtin_fmaf(u, a[lane], r.v0);
                r.k0 = __builtin_fmaf(ds, x[lane], r.k0);
            }
            if (lane + 64 < z.D) {
                r.v1 = __builtin_fmaf(u, a[lane + 64], r.v1);
                r.k1 = __builtin_fmaf(ds, x[lane + 64], r.k1);
            }
        }
    }
    return r;
}
// A query's share of a block of keys; lane d holds dq_d and dq_{d + 64}.
struct QueryPart {
    float q0, q1;
};
__device__ __forceinline__ QueryPart query_part(const Problem& z, const Gradients& g, uint64_t seed, int b, int h, int i, int first,
                                                int end, int lane) {
    QueryPart r{0.0f, 0.0f};
    for (int j0 = first; j0 < first + KEY_BLOCK && j0 < end; j0 += 64) {
        const bool see = seen(z, b, h, i, j0 + lane, end);
        const float mine = pair(z, g, seed, b, h, i, j0 + lane, see).ds;
        const unsigned long long which = __ballot(see);
        for (int n = 0; n < 64; ++n) {
            const float ds = __shfl(mine, n, 64);
            if ((which >> n & 1) == 0) continue;
            const float* x = key_at(z, b, h, j0 + n);
            if (lane < z.D) r.q0 = __builtin_fmaf(ds, x[lane], r.q0);
            if (lane + 64 < z.D) r.q1 = __builtin_fmaf(ds, x[lane + 64], r.q1);
        }
    }
    return r;
}

// Rows in global memory, read and written by offsets in bytes without branches: past `bytes` loads give 0 and stores do nothing. (Rows that
// overlap have others before that end; where they do, `repair` and few_rows leave out by pair what is not seen.)
typedef __amdgpu_buffer_rsrc_t Rows;
constexpr uint32_t NOWHERE = 0xF0000000u;
__device__ __forceinline__ Rows rows_at(const float* base, long long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), (short)0, (int)(bytes > 0 ? bytes : 0), 0x00020000);
}
// `rows` rows (at most 128) of D values, `stride` values apart (at most MAX_ROW).
__device__ __forceinline__ Rows rows_at(const float* base, int rows, long long stride, int D) {
    return rows_at(base, rows > 0 ? ((rows - 1) * stride + D) * 4 : 0);
}
__device__ __forceinline__ float one(Rows r, uint32_t at) { return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0)); }
__device__ __forceinline__ void put_one(Rows r, uint32_t at, float v) {
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), r, at, 0, 0);
}
// Four values from `at` on, of which the first `left` are there. QUADS: 16 bytes at once, all or none there.
template <bool QUADS>
__device__ __forceinline__ float4 four(Rows r, uint32_t at, int left) {
    if (QUADS) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, left > 0 ? at : NOWHERE, 0, 0);
        return make_float4(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3]));
    }
    return make_float4(one(r, left > 0 ? at : NOWHERE), one(r, left > 1 ? at + 4 : NOWHERE), one(r, left > 2 ? at + 8 : NOWHERE),
                       one(r, left > 3 ? at + 12 : NOWHERE));
}
template <bool QUADS>
__device__ __forceinline__ void put_four(Rows r, uint32_t at, int left, const float* v) {
    if (QUADS) {
        typedef uint32_t Words4 __attribute__((ext_vector_type(4)));
        const Words4 w = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
        __builtin_amdgcn_raw_buffer_store_b128(w, r, left > 0 ? at : NOWHERE, 0, 0);
    } else {
#pragma unroll
        for (int n = 0; n < 4; ++n) put_one(r, left > n ? at + 4 * n : NOWHERE, v[n]);
    }
}

// A barrier for what the block's wavefronts hand each other in LDS; loads and stores of global memory may go on across it.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// ---- host ----

constexpr long long MAX_ROW = RG_ATTENTION_MAX_ROW;  // values from a position to the next: 128 positions' offsets stay below 2^31

constexpr long long MAX_BLOCKS = 1 << 23;  // of 256 threads: a launch takes fewer than 2^32

inline unsigned grid_of(long long items, int a_block) {
    const long long blocks = (items + a_block - 1) / a_block;
    return (unsigned)(blocks < 1 ? 1 : blocks < (1 << 20) ? blocks : 1 << 20);
}
// run(DB) with the blocks of 32 values that hold a head's.
template <class F>
void with_size(int D, F run) {
    if (D <= 32) run(std::integral_constant<int, 1>());
    else if (D <= 64) run(std::integral_constant<int, 2>());
    else if (D <= 96) run(std::integral_constant<int, 3>());
    else run(std::integral_constant<int, 4>());
}
template <class F>
void with_flags(bool a, bool b, bool c, F run) {
    const auto third = [&](auto x, auto y) {
        if (c) run(x, y, std::true_type());
        else run(x, y, std::false_type());
    };
    const auto second = [&](auto x) {
        if (b) third(x, std::true_type());
        else third(x, std::false_type());
    };
    if (a) second(std::true_type());
    else second(std::false_type());
}

size_t forward_workspace(const Problem& z, bool masked);  // masked: z's mask will be given
int forward(const Problem& z, float* y, float* stats, unsigned long long* used, void* workspace, hipStream_t stream);
// For at least one query and one key; the workspace starts with the rows' deltas.
size_t backward_workspace(const Problem& z, bool want_bias);
int backward(const Problem& z, const float* dy, const float* stats, float* dq, float* dk, float* dv, float* dbias, void* workspace,
             hipStream_t stream);

}  // namespace attention
}  // namespace rg
