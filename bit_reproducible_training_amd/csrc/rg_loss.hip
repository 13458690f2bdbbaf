// The softmax cross entropy of a vocabulary projection, with its gradients, without keeping the logits.
//
// Tokens are taken in groups (repro_loss::group_tokens), a group's logits z are one product, and its
// gradient dz two more with them: three products in all, where pieces of the vocabulary, whose
// softmax is not known before the last piece, need z a second time.
//
// The matrix cores bound it: of 7.86 ms for 8192 tokens of 768 values against 50257 words (S = 3, four groups, dx and
// dw) the products take 6.24, at 304 TFLOP/s of float32 work, the digits of dz 0.94, the rows' statistics
// 0.36, slicing x and the weight 0.19, the target words 0.07.
#include "rg_digits.h"
#include "rg_internal.h"
#include "repro_loss.h"
#include "repro_loss_math.h"

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace rg {
namespace {

using repro_loss::exp_nonpositive;
using repro_loss::PART;
using repro_loss::Token;

constexpr size_t ALIGN = 256;
size_t align_up(size_t x) { return (x + ALIGN - 1) / ALIGN * ALIGN; }

// 16 bytes at a multiple of 4.
struct __attribute__((packed, aligned(4))) Four {
    float v[4];
};

// What is known of the targets before any product. word: the target, LEFT_OUT or INVALID. A word's
// tokens are listed together from place[word], in ascending order in `list` and as they came in `arrived`.
constexpr int LEFT_OUT = -1, INVALID = -2;
struct Targets {
    int* word;     // [N]
    int* slot;     // [N] the token's place among its word's as they came (which differs from run to run)
    int* arrived;  // [N]
    int* list;     // [N]
    int2* lead;    // [N] of a word's first token: its tokens and their place in `list`; else 0 tokens
    int* count;    // [V]
    int* place;    // [V] (of words that occur)
    int* counted;  // [1] tokens that are not left out
    int* broken;   // [N] 1 where the token's row of x holds a NaN or an infinity (cleared with the rest, set by the slicing)
    int* broken_weight;  // [1] 1 where the weight does
};

// The words' counts by atomics, then places for their tokens. A word's place and its tokens' order in
// `arrived` change from run to run and reach no result: loss_rows puts them in order.
// Each block owns the words of every gridDim.x-th cache line of `count` (gridDim.x a power of two) and reads all targets, so blocks
// need nothing of each other: the places before its own are those of the tokens of the blocks before it. The
// scattered accesses are what takes time, at one compute unit's rate (8192 tokens of 50257 words: 66 us by
// one block, 24 by 16).
// A thread has BATCH tokens in flight. Batches of LISTED tokens come one after another, so a word's tokens of earlier
// batches stand before those of later ones in `arrived`, and only one batch's are left to be ordered.
constexpr int BATCH = 8, LISTED = 1024 * BATCH;
__global__ void __launch_bounds__(1024)
loss_words(const long long* __restrict__ target, long long ignore_index, int N, int V, Targets t) {
    constexpr int threads = 1024, LINE = 32;
    __shared__ int places, kept;
    const int blocks = gridDim.x, self = blockIdx.x;
    // A block's memory operations all meet in its XCD's L2: loads that pass the L1 by, after a barrier that waits
    // for every wavefront's stores and atomics there, see them. (Device-scope fences between the phases
    // write the whole L2 back: 20 us each here.)
    const auto load = [](const int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    const auto phase_end = []() {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    const auto read = [&](int n) {
        const long long v = n < N ? target[n] : ignore_index;
        return v == ignore_index ? LEFT_OUT : v >= 0 && v < V ? (int)v : INVALID;
    };
    if (threadIdx.x == 0) places = kept = 0;
    const int lines = (V + LINE - 1) / LINE;
    for (int i = threadIdx.x; i < (lines - self + blocks - 1) / blocks * LINE; i += threads) {
        const int v = (i / LINE * blocks + self) * LINE + i % LINE;
        if (v < V) t.count[v] = 0;
    }
    phase_end();
    int count = 0, before = 0;
    for (int start = 0; start < N; start += LISTED) {
        const int base = start + threadIdx.x;
        if (start > 0) phase_end();
        int w[BATCH], slot[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) w[i] = read(base + i * threads);
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int owner = w[i] / LINE & (blocks - 1);
            count += w[i] != LEFT_OUT;
            before += w[i] >= 0 && owner < self;
            slot[i] = -1;
            if (w[i] >= 0 && owner == self) slot[i] = atomicAdd(&t.count[w[i]], 1);
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int n = base + i * threads;
            if (n >= N) break;
            if (self == 0) {
                t.word[n] = w[i];
                t.broken[n] = 0;
            }
            if (slot[i] >= 0) t.slot[n] = slot[i];
        }
    }
    if (count > 0) atomicAdd(&kept, count);
    if (before > 0) atomicAdd(&places, before);
    phase_end();
    if (self == 0 && threadIdx.x == 0) {
        t.counted[0] = kept;
        t.broken_weight[0] = 0;
    }
    for (int pass = 0; pass < 2; ++pass) {  // places for the block's words, then its tokens there
        for (int base = threadIdx.x; base < N; base += LISTED) {
            int w[BATCH], slot[BATCH], at[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) w[i] = read(base + i * threads);
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                w[i] = w[i] >= 0 && (w[i] / LINE & (blocks - 1)) == self ? w[i] : LEFT_OUT;
                slot[i] = w[i] >= 0 ? t.slot[base + i * threads] : 0;
                if (pass == 0 && slot[i] > 0) w[i] = LEFT_OUT;
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) at[i] = w[i] >= 0 ? load(pass == 0 ? &t.count[w[i]] : &t.place[w[i]]) : 0;
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                if (w[i] < 0) continue;
                if (pass == 0) t.place[w[i]] = atomicAdd(&places, at[i]);
                else t.arrived[at[i] + slot[i]] = base + i * threads;
            }
        }
        phase_end();
    }
}

// The same for fewer tokens without counts in memory: a token's place is the number of tokens of smaller words, and
// its place among its word's that of earlier ones, so `list` and `lead` are written at once. A block
// takes RANKED tokens, 16 lanes each, which compare them with every token, SHELF at a time from LDS.
constexpr int RANKED = 16, SHELF = 2048;
__global__ void __launch_bounds__(16 * RANKED)
loss_ranks(const long long* __restrict__ target, long long ignore_index, int N, int V, bool lists, Targets t) {
    constexpr int threads = 16 * RANKED;
    __shared__ __align__(16) int shelf[SHELF];
    __shared__ int kept;
    const int l = threadIdx.x & 15, n = blockIdx.x * RANKED + (threadIdx.x >> 4);
    const auto read = [&](int i) {
        const long long v = i < N ? target[i] : ignore_index;
        return v == ignore_index ? LEFT_OUT : v >= 0 && v < V ? (int)v : INVALID;
    };
    const int word = read(n);
    if (threadIdx.x == 0) kept = 0;
    int smaller = 0, same = 0, before = 0, count = 0;
    const bool counts = blockIdx.x == 0;
    for (int first = 0; first < N && (lists || counts); first += SHELF) {
        const int here = min(SHELF, (N - first + 63) / 64 * 64);
        __syncthreads();
        for (int i = threadIdx.x; i < here; i += threads) {
            const int w = read(first + i);
            shelf[i] = w;
            count += w != LEFT_OUT;
        }
        __syncthreads();
        if (!lists) continue;
        for (int i = 4 * l; i < here; i += 64) {
            const int4 four = *reinterpret_cast<const int4*>(&shelf[i]);
            const int w[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                smaller += (uint32_t)w[k] < (uint32_t)word;  // not LEFT_OUT and INVALID: the largest numbers
                same += w[k] == word;
                before += w[k] == word && first + i + k < n;
            }
        }
    }
    if (counts) {
        if (count > 0) atomicAdd(&kept, count);
        __syncthreads();
        if (threadIdx.x == 0) {
            t.counted[0] = kept;
            t.broken_weight[0] = 0;
        }
    }
    if (n >= N) return;
    if (l == 0) {
        t.word[n] = word;
        t.broken[n] = 0;
    }
    if (!lists) return;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) {
        smaller += __shfl_xor(smaller, off, 16);
        same += __shfl_xor(same, off, 16);
        before += __shfl_xor(before, off, 16);
    }
    if (l != 0) return;
    t.lead[n] = make_int2(word >= 0 && before == 0 ? same : 0, smaller);
    if (word >= 0) t.list[smaller + before] = n;
}
// Tokens up to which loss_ranks lists them (us by it and by loss_words: 96 tokens 5.0 and 10.7, 1024 8.5 and 13.8, 2048 13.2
// and 16.8, 4096 19.4 and 19.7, 8192 36.6 and 26.2).
constexpr int RANKS_MAX = 4096;

template <int CTRL>
__device__ __forceinline__ float rotated(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
// Over 16 lanes, in all of them: the tree whose first level joins lanes l and l + 8.
__device__ __forceinline__ float row_sum16(float v) {
    v = v + rotated<0x128>(v);
    v = v + rotated<0x124>(v);
    v = v + rotated<0x122>(v);
    return v + rotated<0x121>(v);
}
__device__ __forceinline__ float row_max16(float v) {
    v = fmaxf(v, rotated<0x128>(v));
    v = fmaxf(v, rotated<0x124>(v));
    v = fmaxf(v, rotated<0x122>(v));
    return fmaxf(v, rotated<0x121>(v));
}
__device__ __forceinline__ float wave_sum(float v) {
    auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return row_sum16(__uint_as_float(s[0]) + __uint_as_float(s[1]));
}

// ---- the logits of few tokens ----
//
// Few tokens' logits are bound by reading the weight once; slicing it first writes 3 bytes for each 4 it reads
// and reads them again. Here a block holds 16 words in registers: its wavefronts take pieces of 64 values of
// each in turn, 16 values of a word a lane, find the words' scales together, round, and contract the digits
// from registers with the tokens' digits, TILES times 16 tokens. The wavefronts' exact integer sums
// meet in LDS. Reading the weight bounds it, at half of HBM's rate, as a block's loads, rounding and products follow
// each other and registers allow few blocks at once. Whole calls without gradients, us, here and by slicing and contracting:
// GPT-2 small's head with 1, 32 and 64 tokens 54, 63 and 92 against 88, 96 and 99; 1600 values a word 115, 134 and 185
// against 180, 186 and 191; 32000 words of 2048 with 32 and 64 tokens 101 and 128 against 146 and 150; 1000 of 256 with
// 8 the same 17. (32 words a block, for one token of GPT-2 small's head 64; registers for 8 pieces where 7 do, for 32
// tokens of 1600 values 153.)
constexpr int FEW_TOKENS = 64, FEW_WAVES = 4, FEW_WORDS_EACH = 16, FEW_K = 2 * PANEL_K, FEW_MAX_D = 8 * FEW_WAVES * FEW_K;
static_assert(STEP_K % FEW_K == 0, "tokens' digits come in whole pieces");

template <int S, int PW, int TILES>
__global__ void __launch_bounds__(64 * FEW_WAVES, PW <= 3 ? 4 : PW <= 4 ? 3 : 2)
loss_few(const float* __restrict__ w, int V, int D, int pieces, const int8_t* __restrict__ qx, const int* __restrict__ ex,
         int N, float* __restrict__ z, int ldz, int* __restrict__ broken_weight) {
    constexpr int L = 2 * S - 1;
    __shared__ int64_t sums[FEW_WAVES][4 * TILES][64];
    __shared__ uint32_t tops[FEW_WAVES][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int word = blockIdx.x * FEW_WORDS_EACH + (lane & 15);
    const float* row = w + (size_t)min(word, V - 1) * D;
    float f[PW][16];
#pragma unroll
    for (int p = 0; p < PW; ++p) {
        const int k0 = (wave + FEW_WAVES * p) * FEW_K + 16 * (lane >> 4);
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            if (k0 + j + 4 <= D) {
                const Four q = *reinterpret_cast<const Four*>(row + k0 + j);
#pragma unroll
                for (int i = 0; i < 4; ++i) f[p][j + i] = q.v[i];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) f[p][j + i] = k0 + j + i < D ? row[k0 + j + i] : 0.0f;
            }
        }
    }
    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < PW; ++p)
#pragma unroll
        for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(f[p][j]) & 0x7FFFFFFFu);
    // (A NaN or an infinity breaks every token: what its word's logits are does not matter.)
    if (top >= 0x7F800000u) broken_weight[0] = 1;
    top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    if (lane < 16) tops[wave][lane] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FEW_WAVES; ++i) top = max(top, tops[i][lane & 15]);
    const int ew = repro_gemm::scale_exponent(__uint_as_float(top));
    const RowScale scale = row_scale<S>(ew);
    v4i acc[TILES][L];
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int l = 0; l < L; ++l) acc[t][l] = v4i{0, 0, 0, 0};
#pragma unroll
    for (int p = 0; p < PW; ++p) {
        // Past the last piece the weight's digits are zero: any of the tokens' will do. A panel is 32 tokens x
        // 32 values, its halves of 16 values one after the other.
        const int8_t* qa = qx + (size_t)min(wave + FEW_WAVES * p, pieces - 1) * (2 * S * PANEL_BYTES) +
                           (lane >> 5) * (S * PANEL_BYTES) + (lane >> 4 & 1) * 512 + (lane & 15) * 16;
        v4i a[TILES][S], b[S];
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int i = 0; i < S; ++i) a[t][i] = *reinterpret_cast<const v4i*>(qa + (size_t)(t >> 1) * pieces * (2 * S * PANEL_BYTES) + i * PANEL_BYTES + (t & 1) * 256);
        int x[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = round_fixed(f[p][j], scale);
        pack16<S>(x, b);
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int j = 0; j < S; ++j)
                    acc[t][i + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[t][i], b[j], acc[t][i + j], 0, 0, 0);
    }
    // Register e of tile t holds token 16 t + 4 (lane / 16) + e and its lane's word.
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            int lv[L];
#pragma unroll
            for (int l = 0; l < L; ++l) lv[l] = acc[t][l][e];
            sums[wave][4 * t + e][lane] = combine_levels<L>(lv);
        }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const int n = 16 * t + 4 * (lane >> 4) + wave;
        int64_t sum = 0;
#pragma unroll
        for (int k = 0; k < FEW_WAVES; ++k) sum += sums[k][4 * t + wave][lane];
        if (n < N && word < V) z[(size_t)n * ldz + word] = round_output(sum, ex[n] + ew - 14 * (S - 1));
    }
}

template <int S, int TILES>
void launch_few_tiles(const float* w, int V, int D, const int8_t* qx, const int* ex, int N, float* z, int ldz, int* broken_weight,
                      hipStream_t st) {
    const int pieces = (D + STEP_K - 1) / STEP_K * (STEP_K / FEW_K);  // as the slicing pads
    const int each = ((D + FEW_K - 1) / FEW_K + FEW_WAVES - 1) / FEW_WAVES;
    decltype(&loss_few<S, 1, TILES>) kernels[] = {loss_few<S, 1, TILES>, loss_few<S, 2, TILES>, loss_few<S, 3, TILES>,
                                                  loss_few<S, 4, TILES>, loss_few<S, 5, TILES>, loss_few<S, 6, TILES>,
                                                  loss_few<S, 7, TILES>, loss_few<S, 8, TILES>};
    hipLaunchKernelGGL(kernels[each - 1], dim3((V + FEW_WORDS_EACH - 1) / FEW_WORDS_EACH), dim3(64 * FEW_WAVES), 0, st, w, V, D, pieces, qx,
                       ex, N, z, ldz, broken_weight);
}
template <int S>
void launch_few_s(const float* w, int V, int D, const int8_t* qx, const int* ex, int N, float* z, int ldz, int* broken_weight,
                  hipStream_t st) {
    if (N <= 16) launch_few_tiles<S, 1>(w, V, D, qx, ex, N, z, ldz, broken_weight, st);
    else if (N <= 32) launch_few_tiles<S, 2>(w, V, D, qx, ex, N, z, ldz, broken_weight, st);
    else launch_few_tiles<S, 4>(w, V, D, qx, ex, N, z, ldz, broken_weight, st);
}

__device__ __forceinline__ float wave_fmax(float m) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    return m;
}

// A token by a block, in one read of its row of z: the parts' largest logits and sums (16 lanes a part, a lane
// a chunk of 4 words, EACH parts in flight), from them the token, its place among its word's (arrived: where
// loss_words has listed them), and the exponent of its row of dz: that of the largest of the words
// other than the target (exp_nonpositive never falls).
// 2047 rows of 50257 take 88 us, 4.7 TB/s, with about 20 vector instructions a logit, the exponential's 13 among
// them, in the same time; 1024 rows 61. By two launches, parts and then tokens, 96 and 67; with the next
// parts in flight 103 and 65; by 512 threads 84 and 61, by 256 87 and 62, but for one token 5 and 15 us more.
// IN_LDS: the parts' maxima and sums are kept there, else in part[row].
// Rows of z are ldz apart, a multiple of 32.
constexpr int EACH = 4, ROW_THREADS = 1024, STRIP = ROW_THREADS / 16;
constexpr int LDS_PARTS = 4096;
static_assert(STRIP == 64, "a wavefront reads the groups' maxima");

template <bool IN_LDS>
__global__ void __launch_bounds__(ROW_THREADS, 8)
loss_rows(const float* __restrict__ z, int ldz, int V, int parts, float2* __restrict__ part, int first, Targets t,
          bool arrived, const float* __restrict__ factors, int mean, Token* __restrict__ tokens,
          int* __restrict__ exponents) {
    extern __shared__ float2 lds_part[];
    __shared__ float maxima[STRIP], others[STRIP];
    __shared__ float target_logit;
    const int r = blockIdx.x, n = first + r, word = t.word[n], lane = threadIdx.x & 63;
    if (word < 0) {  // uniform over the block
        if (threadIdx.x == 0) {
            Token k = repro_loss::ignored_token();
            if (word == INVALID) k.loss = NAN;
            if (arrived) t.lead[n] = make_int2(0, 0);
            tokens[n] = k;
            exponents[r] = 0;
        }
        return;
    }
    float2* kept = IN_LDS ? lds_part : part + (size_t)r * parts;
    const int group = threadIdx.x >> 4, chunk = 4 * (threadIdx.x & 15), own = word / PART;
    const float* q = z + (size_t)r * ldz + chunk;
    float m = -INFINITY, other = -INFINITY;  // other: without the target
    for (int base = group; base < parts; base += STRIP * EACH) {
        float4 f[EACH];
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
            const int at = (base + STRIP * u) * PART;
            f[u] = base + STRIP * u < parts && at + chunk < V ? *reinterpret_cast<const float4*>(q + at) : make_float4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
            const int p = base + STRIP * u, at = p * PART + chunk;
            if (p >= parts) break;  // uniform over a part's 16 lanes
            float v[4] = {f[u].x, f[u].y, f[u].z, f[u].w};
            if (p == parts - 1) {  // words past the last: e^-inf
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = at + i < V ? v[i] : -INFINITY;
            }
            const float a = row_max16(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
            m = fmaxf(m, a);
            float o = a;
            if (p == own) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] = at + i == word ? -INFINITY : v[i];
                    if (at + i == word) target_logit = v[i];
                }
                o = row_max16(fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3])));
            }
            other = fmaxf(other, o);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = v[i] - a;
                v[i] = x >= -87.0f ? repro_loss::exp_in_range(x) : 0.0f;
            }
            // Logits are never NaN (a product is a rounded whole number), so v - a is only where a is infinite, and
            // counted as 0 above: the sum of a part whose logits are all -infinity, while +infinity has none.
            const float b = row_sum16((v[0] + v[1]) + (v[2] + v[3]));
            if (chunk == 0) kept[p] = make_float2(a, a < INFINITY ? b : NAN);
        }
    }
    if (chunk == 0) {
        maxima[group] = m;
        others[group] = other;
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    m = wave_fmax(maxima[lane]);
    other = wave_fmax(others[lane]);
    float s = 0.0f;
    for (int p = lane; p < parts; p += 64) s = s + kept[p].y * exp_nonpositive(kept[p].x - m);
    s = wave_sum(s);
    const float g = factors ? factors[n] : mean ? 1.0f / (float)t.counted[0] : 1.0f;
    const bool broken = t.broken[n] != 0 || t.broken_weight[0] != 0;
    const Token k = broken ? repro_loss::broken_token() : repro_loss::finish_token(m, s, target_logit, g);
    if (arrived) {
        // All of `arrived` that a batch could hold before and after the token's own slot; what stands further before came
        // with an earlier one. (131072 tokens of one word, 256 words of 64 values: 29 ms the call; compared with all of them, 55.)
        const int place = t.place[word], count = t.count[word], slot = t.slot[n];
        const int from = max(0, slot - (LISTED - 1)), to = min(count, slot + LISTED);
        int before = 0;
        for (int i = from + lane; i < to; i += 64) before += t.arrived[place + i] < n;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) before += __shfl_xor(before, off, 64);
        before += from;
        if (lane == 0) {
            t.list[place + before] = n;
            t.lead[n] = make_int2(before == 0 ? count : 0, place);
        }
    }
    if (lane == 0) {
        tokens[n] = k;
        // 0 for a NaN, and a broken token's row of zeros
        exponents[r] = broken ? 0 : repro_gemm::scale_exponent(fabsf(exp_nonpositive(other - k.top) * k.factor));
    }
}

// ---- dz, as the digits that the two products with it read ----
//
// A block takes WORDS words over all of a group's tokens and keeps dz there in registers, so z is
// read once: the words' largest magnitudes, and with them the digits of dz^T for dw, come from there as
// well as the digits of dz for dx, whose tokens' exponents are known. A thread's 4 tokens x 4 words are
// packed along the words and along the tokens; four lanes exchange them into 16-byte pieces of a panel,
// so that a wavefront's stores are whole runs of 1 KiB (rows) and 256 bytes (columns).
// Lane bits 0, 1: q, the words 4 q ..; 2, 3: j, the tokens 16 j ..; 4, 5: i, the tokens 16 j + 4 i ..
constexpr int WORDS = 16, DIGIT_THREADS = 512, STEP_TOKENS = DIGIT_THREADS;  // 64 tokens a wavefront

template <int CTRL>
__device__ __forceinline__ int lane_swapped(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true);
}
// d[k] of lane q becomes d[q] of lane k, among lanes 4 n .. 4 n + 3
__device__ __forceinline__ void transpose_quad(int (&d)[4], int lane) {
    const bool odd = lane & 1, high = lane & 2;
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
        const int got = lane_swapped<0xB1>(odd ? d[k] : d[k + 1]);
        d[k] = odd ? got : d[k];
        d[k + 1] = odd ? d[k + 1] : got;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int got = lane_swapped<0x4E>(high ? d[k] : d[k + 2]);
        d[k] = high ? got : d[k];
        d[k + 2] = high ? d[k + 2] : got;
    }
}
// d[c] of row i of 16 lanes becomes d[i] of row c
__device__ __forceinline__ void transpose_rows(int (&d)[4]) {
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
        const auto s = __builtin_amdgcn_permlane16_swap((uint32_t)d[k], (uint32_t)d[k + 1], false, false);
        d[k] = (int)s[0];
        d[k + 1] = (int)s[1];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const auto s = __builtin_amdgcn_permlane32_swap((uint32_t)d[k], (uint32_t)d[k + 2], false, false);
        d[k] = (int)s[0];
        d[k + 2] = (int)s[1];
    }
}

// round_fixed of a finite value within its row's scale, in the low 7 S bits: the scale is a power of two at least
// |x| / 127 (to one rounding), so |x| 2^n is at most 127 * 2^(7 (S - 1)) when rounded and no clamp is
// needed; what falls below float32's range here rounds to 0 either way.
__device__ __forceinline__ int fixed_bits(float x, int n) {
    return __float_as_int(__builtin_amdgcn_ldexpf(x, n) + ROUND_MAGIC);
}

// Past the caches, which the digits of a group would sweep through before the products read them (2048 tokens of 50257
// words 245 -> 239 us, 1024 121 -> 115; 96 of 1003, whose digits would stay, the same).
__device__ __forceinline__ void store_piece(int8_t* to, const int (&a)[4]) {
    __builtin_nontemporal_store(v4i{a[0], a[1], a[2], a[3]}, reinterpret_cast<v4i*>(to));
}

struct DigitsOut {
    int8_t* by_token;     // op(A) of dx: rows tokens, k words; null where not wanted
    size_t token_bytes;   // of a panel of 32 tokens over all words
    int8_t* by_word;      // op(A) of dw: rows words, k tokens; null where not wanted
    size_t word_bytes;
    int* word_exponents;  // [V]
    int padded;           // the group's tokens, padded as dw's k
};

template <int S, int STEPS>
__global__ void __launch_bounds__(DIGIT_THREADS, 4)
loss_digits(const float* __restrict__ z, int ldz, int V, int first, int rows, const Token* __restrict__ tokens,
            const int* __restrict__ words, const int* __restrict__ exponents, DigitsOut out) {
    __shared__ uint32_t tops[DIGIT_THREADS / 64][WORDS];
    // Neighbouring blocks of words, which share cache lines, run on one XCD (workgroup i on XCD i mod 8).
    const int whole = gridDim.x / 16 * 16, id = blockIdx.x;
    const int block = id < whole ? id / 16 * 16 + id % 8 * 2 + id / 8 % 2 : id;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int q = lane & 3, i = lane >> 4, j = (lane >> 2) & 3;
    const int v0 = block * WORDS, v = v0 + 4 * q;
    const int base = wave * 64 + 16 * j + 4 * i;  // + STEP_TOKENS * step
    float d[STEPS][4][4];
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = s * STEP_TOKENS + base + k;
            const float4 f = r < rows ? *reinterpret_cast<const float4*>(z + (size_t)r * ldz + v) : make_float4(0, 0, 0, 0);
            d[s][k][0] = f.x, d[s][k][1] = f.y, d[s][k][2] = f.z, d[s][k][3] = f.w;
        }
    uint32_t top[4] = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = s * STEP_TOKENS + base + k;
            int word = LEFT_OUT;
            float2 t = make_float2(0.0f, 0.0f);
            if (r < rows) {
                word = words[first + r];
                t = *reinterpret_cast<const float2*>(&tokens[first + r]);  // top, factor (0: a row of zeros)
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float e = repro_loss::dz_of(d[s][k][c], t.x, t.y);
                d[s][k][c] = v + c == word ? 0.0f : e;
                top[c] = max(top[c], __float_as_uint(d[s][k][c]) & 0x7FFFFFFFu);
            }
        }
    if (out.by_token != nullptr) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int t0 = s * STEP_TOKENS + wave * 64;
            if (t0 >= rows) continue;
            v4i w[S];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int r = s * STEP_TOKENS + base + k;
                const int scale = 7 * (S - 1) - (r < rows ? exponents[r] : 0);
                const int x[4] = {fixed_bits(d[s][k][0], scale), fixed_bits(d[s][k][1], scale),
                                  fixed_bits(d[s][k][2], scale), fixed_bits(d[s][k][3], scale)};
                pack_word<S>(x, w, k);
            }
            const int r = s * STEP_TOKENS + base + q;  // the token whose piece this lane stores
            int8_t* to = out.by_token + (size_t)(r >> 5) * out.token_bytes + (size_t)(v0 >> 5) * (S * PANEL_BYTES) +
                         (r & 31) * 16 + (v0 & 16) * 32;
#pragma unroll
            for (int p = 0; p < S; ++p) {
                int a[4] = {w[p][0], w[p][1], w[p][2], w[p][3]};
                transpose_quad(a, lane);
                store_piece(to + p * PANEL_BYTES, a);
            }
        }
    }
    if (out.by_word != nullptr) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int off = 4; off < 64; off <<= 1) top[c] = max(top[c], (uint32_t)__shfl_xor((int)top[c], off, 64));
            if (lane < 4) tops[wave][4 * q + c] = top[c];
        }
        __syncthreads();
        int scale[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t m = 0;
#pragma unroll
            for (int w = 0; w < DIGIT_THREADS / 64; ++w) m = max(m, tops[w][4 * q + c]);
            const int e = repro_gemm::scale_exponent(__uint_as_float(m));
            scale[c] = 7 * (S - 1) - e;
            if (threadIdx.x < 4 && v + c < V) out.word_exponents[v + c] = e;
        }
        const int mine = v0 + 4 * q + i;  // the word whose pieces this lane stores
        int8_t* to = out.by_word + (size_t)(mine >> 5) * out.word_bytes + (mine & 31) * 16;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int t0 = s * STEP_TOKENS + wave * 64;
            if (t0 >= out.padded) continue;
            v4i w[S];  // w[p][c]: digit p of word c's four tokens
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int x[4] = {fixed_bits(d[s][0][c], scale[c]), fixed_bits(d[s][1][c], scale[c]),
                                  fixed_bits(d[s][2][c], scale[c]), fixed_bits(d[s][3][c], scale[c])};
                pack_word<S>(x, w, c);
            }
            const int k0 = t0 + 16 * j;
#pragma unroll
            for (int p = 0; p < S; ++p) {
                int a[4] = {w[p][0], w[p][1], w[p][2], w[p][3]};
                transpose_rows(a);
                store_piece(to + ((size_t)(k0 >> 5) * S + p) * PANEL_BYTES + (k0 & 16) * 32, a);
            }
        }
    }
}

// The sum or mean of the losses, by a block.
template <int THREADS>
__device__ __forceinline__ void reduce_losses(const Token* __restrict__ tokens, int N, int reduction,
                                              const int* __restrict__ counted, float* __restrict__ loss) {
    constexpr int OWN = repro_loss::STRANDS / THREADS;
    __shared__ double lds[repro_loss::STRANDS];
    double s[OWN];
#pragma unroll
    for (int k = 0; k < OWN; ++k) s[k] = 0.0;
#pragma unroll 4
    for (int base = 0; base < N; base += repro_loss::STRANDS) {
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
            const int n = base + k * THREADS + threadIdx.x;
            if (n < N) s[k] = s[k] + (double)tokens[n].loss;
        }
    }
#pragma unroll
    for (int k = 0; k < OWN; ++k) lds[k * THREADS + threadIdx.x] = s[k];
    for (int h = repro_loss::STRANDS / 2; h > 0; h /= 2) {
        __syncthreads();
        for (int i = threadIdx.x; i < h; i += THREADS) lds[i] = lds[i] + lds[i + h];
    }
    if (threadIdx.x == 0) loss[0] = (float)(reduction == RG_LOSS_MEAN ? lds[0] / (double)counted[0] : lds[0]);
}

// ---- the target words' share ----
//
// A wavefront takes a token and 256 columns, of dx (blockIdx.z 0) or of dw, where a word's first token
// stands for all of its tokens, 16 at a time. Most words have one, whose row's address is known without the list.
// loss: where the losses' sum or mean is wanted, the first block of the launch takes it (a launch of its own: 5 us), and
// the tokens start with the second.
__global__ void __launch_bounds__(256)
loss_target(float* __restrict__ dx, float* __restrict__ dw, const float* __restrict__ x, const float* __restrict__ w,
            int D, const Token* __restrict__ tokens, Targets t, int N, int reduction, float* __restrict__ loss) {
    if (loss != nullptr && blockIdx.x == 0) {
        if (blockIdx.y == 0 && blockIdx.z == 0) reduce_losses<256>(tokens, N, reduction, t.counted, loss);
        return;
    }
    const int lane = threadIdx.x & 63;
    const int n = (blockIdx.x - (loss != nullptr)) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int at = blockIdx.y * 256 + 4 * lane;
    if (n >= N || at >= D) return;
    const bool full = at + 4 <= D;
    const auto load = [&](const float* p, float (&v)[4]) {
        if (full) {
            const Four f = *reinterpret_cast<const Four*>(p + at);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = f.v[k];
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = at + k < D ? p[at + k] : 0.0f;
        }
    };
    const auto onto = [&](float* p, const float (&v)[4]) {
        float old[4];
        load(p, old);
        Four f;
#pragma unroll
        for (int k = 0; k < 4; ++k) f.v[k] = old[k] + v[k];
        if (full) {
            *reinterpret_cast<Four*>(p + at) = f;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (at + k < D) p[at + k] = f.v[k];
        }
    };
    const int word = t.word[n];
    const float mine = tokens[n].target;
    float v[4];
    if (blockIdx.z == 0 && dx != nullptr) {
        if (word < 0) return;
        load(w + (size_t)word * D, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = mine * v[k];
        onto(dx + (size_t)n * D, v);
        return;
    }
    const int2 lead = t.lead[n];
    if (lead.x == 0) return;
    if (lead.x == 1) {
        load(x + (size_t)n * D, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = 0.0f + mine * v[k];
        onto(dw + (size_t)word * D, v);
        return;
    }
    const int* list = t.list + lead.y;
    float s[16][4];
#pragma unroll
    for (int h = 0; h < 16; ++h)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[h][k] = 0.0f;
    for (int k0 = 0; k0 < lead.x; k0 += 16) {
        // No branches: the 16 rows are in flight together (past the end the last one, whose value is not taken).
        float c[16], q[16][4];
#pragma unroll
        for (int h = 0; h < 16; ++h) {
            const int m = list[min(k0 + h, lead.x - 1)];
            c[h] = tokens[m].target;
            load(x + (size_t)m * D, q[h]);
        }
#pragma unroll
        for (int h = 0; h < 16; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[h][k] = k0 + h < lead.x ? s[h][k] + c[h] * q[h][k] : s[h][k];
    }
#pragma unroll
    for (int h = 8; h > 0; h /= 2)
#pragma unroll
        for (int a = 0; a < h; ++a)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[a][k] = s[a][k] + s[a + h][k];
    onto(dw + (size_t)word * D, s[0]);
}

// The losses, or their sum or mean (one block).
__global__ void __launch_bounds__(1024)
loss_reduce(const Token* __restrict__ tokens, int N, int reduction, const int* __restrict__ counted, float* __restrict__ loss) {
    if (reduction != RG_LOSS_NONE) return reduce_losses<1024>(tokens, N, reduction, counted, loss);
    for (int n = blockIdx.x * 1024 + threadIdx.x; n < N; n += gridDim.x * 1024) loss[n] = tokens[n].loss;
}

__global__ void __launch_bounds__(256) loss_fill(float* __restrict__ a, float v, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) a[i] = v;
}
__device__ __forceinline__ void scale_all(float* __restrict__ a, size_t n, float f) {
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x, all = (size_t)gridDim.x * 256;
    for (size_t i = id; i < n / 4; i += all) {
        Four v = reinterpret_cast<Four*>(a)[i];
#pragma unroll
        for (int k = 0; k < 4; ++k) v.v[k] = v.v[k] * f;
        reinterpret_cast<Four*>(a)[i] = v;
    }
    if (id < n % 4) a[n - 1 - id] = a[n - 1 - id] * f;
}
__global__ void __launch_bounds__(256)
scale_kernel(float* __restrict__ a, size_t na, float* __restrict__ b, size_t nb, const float* __restrict__ factor) {
    const float f = factor[0];
    if (f == 1.0f) return;
    scale_all(a, na, f);
    scale_all(b, nb, f);
}

unsigned grid_of(size_t n) { return (unsigned)std::min<size_t>((n + 255) / 256, 1u << 20); }

bool sizes_ok(const rg_loss_config* c) {
    return c && c->N >= 0 && c->N <= RG_LOSS_MAX_TOKENS && c->D >= 1 && c->D <= RG_LOSS_MAX_SIZE && c->V >= 1 &&
           c->V <= RG_LOSS_MAX_WORDS && c->slices >= 1 && c->slices <= 3 &&
           c->reduction >= RG_LOSS_MEAN && c->reduction <= RG_LOSS_NONE;
}

int round_up(int x, int m) { return (x + m - 1) / m * m; }

// A product from digits that are in memory: the tile plan (no kernel that slices by itself).
int plan_product(int M, int N, int K, int S, Layout* L) {
    rg_config c;
    rg_config_init(&c);
    c.slices = S;
    PlanExtras extras;
    extras.one_launch = false;
    return layout_for_current_device(M, N, K, &c, L, extras);
}

struct Digits {
    size_t q, e;  // offsets of the panels and exponents
};

// Where everything lies in the workspace, and the products of a whole group [0] and of the last [1].
struct Space {
    int group, last, parts, ldz;
    bool few;  // the logits by loss_few
    Layout z[2], dx[2], dw[2];
    Digits x_rows, w_rows, w_cols, x_cols, by_token, by_word;
    size_t words, tokens, part, logits, partial, scratch, total;
};

int plan_space(const rg_loss_config* c, bool dx, bool dw, Space* s) {
    const int N = (int)c->N, D = c->D, V = c->V, S = c->slices;
    s->group = std::min(repro_loss::group_tokens(V), N);
    s->last = (N - 1) % s->group + 1;
    s->parts = (V + PART - 1) / PART;
    s->ldz = round_up(V, 32);
    s->few = N <= FEW_TOKENS && D <= FEW_MAX_D;
    // Rows past a matrix's own that a tile may read: their products are not stored.
    constexpr int BEYOND = 192;
    size_t at = 0, partial = 0, scratch = 0;
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align_up(bytes);
        return here;
    };
    const auto digits = [&](int rows, int K) {
        Digits d;
        d.q = take((size_t)(round_up(rows, 64) + BEYOND) * round_up(K, STEP_K) * S);
        d.e = take((size_t)(round_up(rows, 64) + BEYOND) * sizeof(int));
        return d;
    };
    for (int k = 0; k < 2; ++k) {
        const int rows = k ? s->last : s->group;
        int rc = s->few ? hipSuccess : plan_product(rows, V, D, S, &s->z[k]);
        if (rc == hipSuccess && dx) rc = plan_product(rows, D, V, S, &s->dx[k]);
        if (rc == hipSuccess && dw) rc = plan_product(V, D, rows, S, &s->dw[k]);
        if (rc != hipSuccess) return rc;
        for (const Layout* L : {s->few ? nullptr : &s->z[k], dx ? &s->dx[k] : nullptr, dw ? &s->dw[k] : nullptr})
            if (L && L->has_partial) partial = std::max(partial, (size_t)L->split * L->M * L->N * sizeof(int64_t));
    }
    s->words = take(((size_t)7 * N + 2 * (size_t)round_up(V, 32) + 2) * sizeof(int));
    s->tokens = take((size_t)N * sizeof(Token));
    s->part = take(s->parts <= LDS_PARTS ? 0 : (size_t)s->group * s->parts * sizeof(float2));
    s->logits = take((size_t)s->group * s->ldz * sizeof(float));
    s->x_rows = digits(N, D);
    s->w_rows = digits(s->few ? 0 : V, D);
    scratch = std::max(slice_scratch_bytes(N, D, false), slice_scratch_bytes(V, D, false));
    if (dx) {
        s->w_cols = digits(D, V);
        scratch = std::max(scratch, slice_scratch_bytes(D, V, true));
    }
    s->by_token = digits(s->group, dx ? V : 0);
    if (dw) {
        s->x_cols = digits(D, s->group);
        scratch = std::max({scratch, slice_scratch_bytes(D, s->group, true), slice_scratch_bytes(D, s->last, true)});
        s->by_word = digits(V, s->group);
    }
    s->partial = take(partial);
    s->scratch = take(scratch);
    s->total = at;
    return hipSuccess;
}

// C (rows ldc apart) = the product of two operands' digits, or that added to C.
void launch_product(const Layout& L, const int8_t* qa, const int* ea, const int8_t* qb, const int* eb, float* C,
                    long long ldc, bool onto, int64_t* partial, hipStream_t st) {
    const OutAddr out{ldc, 0, nullptr, onto};
    launch_contract_mfma(L, qa, qb, ea, eb, C, out, L.has_partial ? partial : nullptr, st);
    if (L.has_partial) launch_reduce_round(L, partial, ea, eb, C, out, st);
}

template <int S>
void launch_digits_s(int V, int rows, hipStream_t st, const float* z, int ldz, int first, const Token* tokens,
                     const int* words, const int* exponents, const DigitsOut& out) {
    const dim3 grid((V + WORDS - 1) / WORDS), block(DIGIT_THREADS);
    auto kernel = rows <= STEP_TOKENS ? loss_digits<S, 1> : rows <= 2 * STEP_TOKENS ? loss_digits<S, 2> : loss_digits<S, 4>;
    hipLaunchKernelGGL(kernel, grid, block, 0, st, z, ldz, V, first, rows, tokens, words, exponents, out);
}
static_assert(repro_loss::MAX_GROUP <= 4 * STEP_TOKENS, "a block holds a group's tokens");
static_assert(repro_loss::MAX_GROUP <= ONEPASS_MAX_K_COLUMNS && sizeof(Token) == 4 * sizeof(float),
              "a group's tokens are sliced in one pass, which reads their factors");

}  // namespace
}  // namespace rg

extern "C" {

void rg_loss_config_init(rg_loss_config* cfg) {
    if (!cfg) return;
    cfg->N = 0;
    cfg->D = cfg->V = 0;
    cfg->slices = 3;
    cfg->reduction = RG_LOSS_MEAN;
    cfg->ignore_index = -100;
}

int rg_loss_group_tokens(int V) { return V < 1 ? 0 : repro_loss::group_tokens(V); }

int rg_linear_cross_entropy_workspace(const rg_loss_config* cfg, int want_dx, int want_dw, size_t* bytes) {
    if (!rg::sizes_ok(cfg) || !bytes) return hipErrorInvalidValue;
    *bytes = 0;
    if (cfg->N == 0) return hipSuccess;
    rg::Space s;
    const int rc = rg::plan_space(cfg, want_dx != 0, want_dw != 0, &s);
    if (rc == hipSuccess) *bytes = s.total;
    return rc;
}

int rg_linear_cross_entropy(const rg_loss_config* cfg, const float* x, const float* w, const long long* target,
                            const float* factors, float* loss, float* dx, float* dw, void* workspace,
                            size_t workspace_bytes, void* stream) {
    using namespace rg;
    if (!sizes_ok(cfg)) return hipErrorInvalidValue;
    const auto off = [](const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; };
    if (off(x, 4) || off(w, 4) || off(target, 8) || off(factors, 4) || off(loss, 4) || off(dx, 4) || off(dw, 4))
        return hipErrorInvalidValue;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int D = cfg->D, V = cfg->V, N = (int)cfg->N, S = cfg->slices;
    if (N == 0) {
        if (!dw && (!loss || cfg->reduction == RG_LOSS_NONE)) return hipSuccess;
        const auto fill = [&](float* p, float v, size_t n) {
            if (p) hipLaunchKernelGGL(loss_fill, dim3(grid_of(n)), dim3(256), 0, st, p, v, n);
        };
        if (cfg->reduction != RG_LOSS_NONE) fill(loss, cfg->reduction == RG_LOSS_MEAN ? NAN : 0.0f, 1);
        fill(dw, 0.0f, (size_t)V * D);
        return hipGetLastError();
    }
    if (!x || !w || !target) return hipErrorInvalidValue;
    Space s;
    int rc = plan_space(cfg, dx != nullptr, dw != nullptr, &s);
    if (rc != hipSuccess) return rc;
    if (!workspace || off(workspace, 256) || workspace_bytes < s.total) return hipErrorInvalidValue;
    char* base = static_cast<char*>(workspace);
    const auto panels = [&](const Digits& d) { return reinterpret_cast<int8_t*>(base + d.q); };
    const auto exponents = [&](const Digits& d) { return reinterpret_cast<int*>(base + d.e); };
    Targets t;
    t.count = reinterpret_cast<int*>(base + s.words);  // whole cache lines
    t.place = t.count + round_up(V, 32);
    t.lead = reinterpret_cast<int2*>(t.place + round_up(V, 32));
    t.word = reinterpret_cast<int*>(t.lead + N);
    t.slot = t.word + N;
    t.arrived = t.slot + N;
    t.list = t.arrived + N;
    t.counted = t.list + N;
    t.broken_weight = t.counted + 1;
    t.broken = t.broken_weight + 1;
    Token* tokens = reinterpret_cast<Token*>(base + s.tokens);
    float2* part = reinterpret_cast<float2*>(base + s.part);
    float* z = reinterpret_cast<float*>(base + s.logits);
    int64_t* partial = reinterpret_cast<int64_t*>(base + s.partial);
    float* scratch = reinterpret_cast<float*>(base + s.scratch);

    const bool ranked = !dw || N <= RANKS_MAX;
    if (ranked)
        hipLaunchKernelGGL(loss_ranks, dim3((N + RANKED - 1) / RANKED), dim3(16 * RANKED), 0, st, target, cfg->ignore_index,
                           N, V, dw != nullptr, t);
    else
        hipLaunchKernelGGL(loss_words, dim3(16), dim3(1024), 0, st, target, cfg->ignore_index, N, V, t);
    // The digits that every group's products share.
    rc = launch_slice_rows(x, N, panels(s.x_rows), exponents(s.x_rows), t.broken, s.few ? nullptr : w, V, panels(s.w_rows),
                           exponents(s.w_rows), t.broken_weight, D, S, scratch, st);
    if (rc == hipSuccess && dx) rc = launch_slice(w, D, V, true, S, panels(s.w_cols), exponents(s.w_cols), scratch, st);
    if (rc != hipSuccess) return rc;
    for (int first = 0; first < N; first += s.group) {
        const int rows = std::min(s.group, N - first), k = first + s.group < N ? 0 : 1;
        if (s.few) {
            auto launch_few = S == 1 ? launch_few_s<1> : S == 2 ? launch_few_s<2> : launch_few_s<3>;
            launch_few(w, V, D, panels(s.x_rows), exponents(s.x_rows), N, z, s.ldz, t.broken_weight, st);
        } else {
            launch_product(s.z[k], panels(s.x_rows) + (size_t)first * round_up(D, STEP_K) * S, exponents(s.x_rows) + first,
                           panels(s.w_rows), exponents(s.w_rows), z, s.ldz, false, partial, st);
        }
        const bool in_lds = s.parts <= LDS_PARTS;
        hipLaunchKernelGGL(in_lds ? loss_rows<true> : loss_rows<false>, dim3(rows), dim3(ROW_THREADS),
                           in_lds ? s.parts * sizeof(float2) : 0, st, z, s.ldz, V, s.parts, part, first, t, !ranked, factors,
                           cfg->reduction == RG_LOSS_MEAN ? 1 : 0, tokens, exponents(s.by_token));
        if (!dx && !dw) continue;
        DigitsOut out;
        out.by_token = dx ? panels(s.by_token) : nullptr;
        out.token_bytes = (size_t)round_up(V, STEP_K) * S * PANEL_ROWS;
        out.padded = round_up(rows, STEP_K);
        out.by_word = dw ? panels(s.by_word) : nullptr;
        out.word_bytes = (size_t)out.padded * S * PANEL_ROWS;
        out.word_exponents = dw ? exponents(s.by_word) : nullptr;
        if (S == 1) launch_digits_s<1>(V, rows, st, z, s.ldz, first, tokens, t.word, exponents(s.by_token), out);
        else if (S == 2) launch_digits_s<2>(V, rows, st, z, s.ldz, first, tokens, t.word, exponents(s.by_token), out);
        else launch_digits_s<3>(V, rows, st, z, s.ldz, first, tokens, t.word, exponents(s.by_token), out);
        if (dx)
            launch_product(s.dx[k], panels(s.by_token), exponents(s.by_token), panels(s.w_cols), exponents(s.w_cols),
                           dx + (size_t)first * D, D, false, partial, st);
        if (dw) {
            rc = launch_slice(x + (size_t)first * D, D, rows, true, S, panels(s.x_cols), exponents(s.x_cols), scratch, st,
                              &tokens[first].factor);
            if (rc != hipSuccess) return rc;
            launch_product(s.dw[k], panels(s.by_word), exponents(s.by_word), panels(s.x_cols), exponents(s.x_cols),
                           dw, D, first > 0, partial, st);
        }
    }
    const bool joined = loss && cfg->reduction != RG_LOSS_NONE && (dx || dw);
    if (dx || dw)
        hipLaunchKernelGGL(loss_target, dim3((N + 3) / 4 + joined, (D + 255) / 256, dx && dw ? 2 : 1), dim3(256), 0, st, dx,
                           dw, x, w, D, tokens, t, N, cfg->reduction, joined ? loss : nullptr);
    if (loss && !joined)
        hipLaunchKernelGGL(loss_reduce, dim3(cfg->reduction == RG_LOSS_NONE ? std::min((N + 1023) / 1024, 1024) : 1),
                           dim3(1024), 0, st, tokens, N, cfg->reduction, t.counted, loss);
    return hipGetLastError();
}

int rg_scale_fp32(float* x, size_t nx, float* y, size_t ny, const float* factor, void* stream) {
    if (nx + ny == 0) return hipSuccess;
    if ((nx > 0 && !x) || (ny > 0 && !y) || !factor) return hipErrorInvalidValue;
    const unsigned grid = (unsigned)std::min<size_t>((nx + ny + 1023) / 1024, 4096);
    hipLaunchKernelGGL(rg::scale_kernel, dim3(grid), dim3(256), 0, static_cast<hipStream_t>(stream), x, nx, y, ny, factor);
    return hipGetLastError();
}

}  // extern "C"
