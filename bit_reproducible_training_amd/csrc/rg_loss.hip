// The softmax cross entropy of a vocabulary projection, with its gradients, without keeping the logits.
//
// Tokens are taken in groups (repro_loss::group_tokens), a group's logits z are one product, and its
// gradient dz two more with them: three products in all, where pieces of the vocabulary, whose
// softmax is not known before the last piece, need z a second time.
#include "rg_internal.h"
#include "repro_loss.h"
#include "repro_loss_math.h"
#include "repro_sum.h"

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

// What is known of the targets before any product. word: the target, LEFT_OUT or INVALID. The tokens
// of a word are listed together in ascending order, from place[first token of the word].
constexpr int LEFT_OUT = -1, INVALID = -2;
struct Targets {
    int* word;    // [N]
    int* first;   // [N] the first token of its word
    int* rank;    // [N] its word's tokens before it
    int* count;   // [N] its word's tokens (where rank is 0)
    int* place;   // [N] (where rank is 0)
    int* list;    // [N]
    int* used;    // places given out, tokens that count
};

__global__ void loss_clear(int* used) { used[0] = used[1] = 0; }

// A wavefront takes a token and compares its word with every token's, which the block's 16
// wavefronts read through LDS together.
constexpr int WORDS_THREADS = 1024, WORDS_TILE = 4096;
__global__ void __launch_bounds__(WORDS_THREADS)
loss_words(const long long* __restrict__ target, long long ignore_index, int N, int V, Targets t) {
    __shared__ int tile[WORDS_TILE];
    const int lane = threadIdx.x & 63;
    const int n = blockIdx.x * (WORDS_THREADS / 64) + (threadIdx.x >> 6);
    const auto read = [&](int i) {
        const long long v = target[i];
        return v == ignore_index ? LEFT_OUT : v >= 0 && v < V ? (int)v : INVALID;
    };
    const int mine = n < N ? read(n) : LEFT_OUT;
    int before = 0, all = 0, first = N;
    for (int base = 0; base < N; base += WORDS_TILE) {
        __syncthreads();
        for (int i = threadIdx.x; i < WORDS_TILE && base + i < N; i += WORDS_THREADS) tile[i] = read(base + i);
        __syncthreads();
        const int held = min(WORDS_TILE, N - base);
        for (int i = lane; i < held; i += 64) {
            const bool same = tile[i] == mine;
            all += same;
            before += same && base + i < n;
            first = same ? min(first, base + i) : first;
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        all += __shfl_xor(all, off, 64);
        before += __shfl_xor(before, off, 64);
        first = min(first, __shfl_xor(first, off, 64));
    }
    if (lane != 0 || n >= N) return;
    t.word[n] = mine;
    t.rank[n] = before;
    t.first[n] = first;
    if (mine >= 0 && before == 0) {
        t.count[n] = all;
        t.place[n] = atomicAdd(&t.used[0], all);  // which place a word gets changes no result
    }
    if (mine != LEFT_OUT) atomicAdd(&t.used[1], 1);
}

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

// The parts' largest logits and sums: a lane takes a chunk of 4 words, 16 lanes a part.
__global__ void __launch_bounds__(256)
loss_parts(const float* __restrict__ z, int V, int parts, float2* __restrict__ out) {
    const int row = blockIdx.y;
    const int part = blockIdx.x * 16 + (threadIdx.x >> 4);
    if (part >= parts) return;  // uniform over a part's 16 lanes
    const int at = part * PART + 4 * (threadIdx.x & 15);
    const float* q = z + (size_t)row * V;
    float v[4];
    if (at + 4 <= V) {
        const Four f = *reinterpret_cast<const Four*>(q + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = f.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = at + i < V ? q[at + i] : -INFINITY;
    }
    const float a = row_max16(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = at + i < V ? exp_nonpositive(v[i] - a) : 0.0f;
    const float b = row_sum16((v[0] + v[1]) + (v[2] + v[3]));
    if ((threadIdx.x & 15) == 0) out[(size_t)row * parts + part] = make_float2(a, b);
}

// A token from its parts (a wavefront each), and its place in its word's list.
__global__ void __launch_bounds__(256)
loss_tokens(const float* __restrict__ z, int V, int parts, const float2* __restrict__ part, int first, int rows,
            Targets t, const float* __restrict__ factors, int mean, Token* __restrict__ tokens,
            float* __restrict__ losses) {
    const int lane = threadIdx.x & 63;
    const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    const int n = first + r, word = t.word[n];
    Token k = repro_loss::ignored_token();
    if (word >= 0) {
        const float2* p = part + (size_t)r * parts;
        float m = -INFINITY;
        for (int i = lane; i < parts; i += 64) m = fmaxf(m, p[i].x);
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        float s = 0.0f;
        for (int i = lane; i < parts; i += 64) s = s + p[i].y * exp_nonpositive(p[i].x - m);
        s = wave_sum(s);
        const float g = factors ? factors[n] : mean ? 1.0f / (float)t.used[1] : 1.0f;
        k = repro_loss::finish_token(m, s, z[(size_t)r * V + word], g);
        if (lane == 0) t.list[t.place[t.first[n]] + t.rank[n]] = n;
    } else if (word == INVALID) {
        k.loss = NAN;
    }
    if (lane == 0) {
        tokens[n] = k;
        losses[n] = k.loss;
    }
}

// z becomes its gradient, without the target words' share.
__global__ void __launch_bounds__(256)
loss_gradient(float* __restrict__ z, int V, int first, const Token* __restrict__ tokens, const int* __restrict__ words) {
    const int row = blockIdx.y;
    const Token k = tokens[first + row];
    const int word = words[first + row];
    float* q = z + (size_t)row * V;
    const int at = 4 * (blockIdx.x * 256 + threadIdx.x);
    if (at >= V) return;
    Four f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = at + i < V ? q[at + i] : 0.0f;
        f.v[i] = word < 0 || at + i == word ? 0.0f : exp_nonpositive(v - k.top) * k.factor;
    }
    if (at + 4 <= V) *reinterpret_cast<Four*>(q + at) = f;
    else
        for (int i = 0; i < 4; ++i)
            if (at + i < V) q[at + i] = f.v[i];
}

// The target words' share of dx.
__global__ void __launch_bounds__(256)
loss_target_dx(float* __restrict__ dx, const float* __restrict__ w, int D, const Token* __restrict__ tokens,
               const int* __restrict__ words, int N) {
    for (int n = blockIdx.x; n < N; n += gridDim.x) {
        const int word = words[n];
        if (word < 0) continue;
        const float c = tokens[n].target;
        const float* q = w + (size_t)word * D;
        float* o = dx + (size_t)n * D;
        for (int i = threadIdx.x; i < D; i += 256) o[i] = o[i] + c * q[i];
    }
}

// The target words' share of dw: a block takes a word (at its first token), a wavefront 256 columns
// at a time, 16 of the word's tokens in flight.
__global__ void __launch_bounds__(256)
loss_target_dw(float* __restrict__ dw, const float* __restrict__ x, int D, const Token* __restrict__ tokens, Targets t,
               int N) {
    const int n = blockIdx.x, word = t.word[n];
    if (word < 0 || t.rank[n] != 0) return;
    const int count = t.count[n];
    const int* list = t.list + t.place[n];
    const int lane = threadIdx.x & 63;
    for (int base = 256 * (threadIdx.x >> 6); base < D; base += 1024) {
        const int at = base + 4 * lane;
        float s[16][4];
#pragma unroll
        for (int h = 0; h < 16; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[h][i] = 0.0f;
        for (int k0 = 0; k0 < count; k0 += 16) {
#pragma unroll
            for (int h = 0; h < 16; ++h) {
                if (k0 + h >= count) break;
                const int m = list[k0 + h];
                const float c = tokens[m].target;
                const float* q = x + (size_t)m * D;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at + i < D) s[h][i] = s[h][i] + c * q[at + i];
            }
        }
#pragma unroll
        for (int h = 8; h > 0; h /= 2)
#pragma unroll
            for (int k = 0; k < h; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[k][i] = s[k][i] + s[k + h][i];
        float* o = dw + (size_t)word * D;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i < D) o[at + i] = o[at + i] + s[0][i];
    }
}

__global__ void __launch_bounds__(256) loss_add(float* __restrict__ a, const float* __restrict__ b, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) a[i] = a[i] + b[i];
}
__global__ void __launch_bounds__(256) loss_fill(float* __restrict__ a, float v, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) a[i] = v;
}
__global__ void __launch_bounds__(256) scale_kernel(float* __restrict__ a, const float* __restrict__ factor, size_t n) {
    const float f = factor[0];
    if (f == 1.0f) return;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) a[i] = a[i] * f;
}
__global__ void loss_mean(float* loss, const int* used) { loss[0] = loss[0] / (float)used[1]; }

unsigned grid_of(size_t n) { return (unsigned)std::min<size_t>((n + 255) / 256, 1u << 20); }

bool sizes_ok(const rg_loss_config* c) {
    return c && c->N >= 0 && c->N <= 2147483647ll && c->D >= 1 && c->V >= 1 && c->slices >= 1 && c->slices <= 3 &&
           c->reduction >= RG_LOSS_MEAN && c->reduction <= RG_LOSS_NONE;
}

rg_config product(int slices, bool ta, bool tb) {
    rg_config g;
    rg_config_init(&g);
    g.slices = slices;
    g.trans_a = ta;
    g.trans_b = tb;
    return g;
}

// Where everything lies in the workspace.
struct Space {
    int group, parts;
    size_t words, tokens, losses, part, z, dw, gemm, sum, gemm_bytes, sum_bytes, total;
};

int plan_space(const rg_loss_config* c, bool dx, bool dw, Space* s) {
    const size_t N = (size_t)c->N;
    s->group = (int)std::min<long long>(repro_loss::group_tokens(c->V), c->N);
    s->parts = (c->V + PART - 1) / PART;
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align_up(bytes);
        return here;
    };
    s->words = take((6 * N + 2) * sizeof(int));
    s->tokens = take(N * sizeof(Token));
    s->losses = take(N * sizeof(float));
    s->part = take((size_t)s->group * s->parts * sizeof(float2));
    s->z = take((size_t)s->group * c->V * sizeof(float));
    s->dw = take(dw && c->N > s->group ? (size_t)c->V * c->D * sizeof(float) : 0);
    s->gemm_bytes = s->sum_bytes = 0;
    const auto need = [&](int M, int N_, int K, bool ta, bool tb) {
        const rg_config g = product(c->slices, ta, tb);
        rg_plan p;
        const int rc = rg_make_plan(M, N_, K, &g, &p);
        if (rc == hipSuccess) s->gemm_bytes = std::max(s->gemm_bytes, p.workspace_bytes);
        return rc;
    };
    // a whole group and the last one
    for (const int rows : {s->group, c->N > 0 ? (int)((c->N - 1) % s->group) + 1 : 0}) {
        if (rows == 0) continue;
        int rc = need(rows, c->V, c->D, false, true);
        if (rc == hipSuccess && dx) rc = need(rows, c->D, c->V, false, false);
        if (rc == hipSuccess && dw) rc = need(c->V, c->D, rows, true, false);
        if (rc != hipSuccess) return rc;
    }
    s->gemm = take(s->gemm_bytes);
    if (c->N > 0 && c->reduction != RG_LOSS_NONE) {
        rg_sum_config sc;
        rg_sum_config_init(&sc);
        rg_sum_plan p;
        const int rc = rg_make_sum_plan(1, 1, (int)c->N, &sc, &p);
        if (rc != hipSuccess) return rc;
        s->sum_bytes = p.workspace_bytes;
    }
    s->sum = take(s->sum_bytes);
    s->total = at;
    return hipSuccess;
}

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
    const int D = cfg->D, V = cfg->V, N = (int)cfg->N;
    const auto fill = [&](float* p, float v, size_t n) {
        if (p) hipLaunchKernelGGL(loss_fill, dim3(grid_of(n)), dim3(256), 0, st, p, v, n);
    };
    if (N == 0) {
        if (!dw && (!loss || cfg->reduction == RG_LOSS_NONE)) return hipSuccess;
        if (cfg->reduction != RG_LOSS_NONE) fill(loss, cfg->reduction == RG_LOSS_MEAN ? NAN : 0.0f, 1);
        fill(dw, 0.0f, (size_t)V * D);
        return hipGetLastError();
    }
    if (!x || !w || !target) return hipErrorInvalidValue;
    Space s;
    int rc = plan_space(cfg, dx != nullptr, dw != nullptr, &s);
    if (rc != hipSuccess) return rc;
    if (!workspace || off(workspace, 16) || workspace_bytes < s.total) return hipErrorInvalidValue;
    char* base = static_cast<char*>(workspace);
    Targets t;
    t.word = reinterpret_cast<int*>(base + s.words);
    t.first = t.word + N;
    t.rank = t.first + N;
    t.count = t.rank + N;
    t.place = t.count + N;
    t.list = t.place + N;
    t.used = t.list + N;
    Token* tokens = reinterpret_cast<Token*>(base + s.tokens);
    float* losses = reinterpret_cast<float*>(base + s.losses);
    float2* part = reinterpret_cast<float2*>(base + s.part);
    float* z = reinterpret_cast<float*>(base + s.z);
    float* more = reinterpret_cast<float*>(base + s.dw);
    hipLaunchKernelGGL(loss_clear, dim3(1), dim3(1), 0, st, t.used);
    hipLaunchKernelGGL(loss_words, dim3((N + 15) / 16), dim3(WORDS_THREADS), 0, st, target, cfg->ignore_index, N, V, t);
    for (int first = 0; first < N; first += s.group) {
        const int rows = std::min(s.group, N - first);
        const float* xg = x + (size_t)first * D;
        rg_config g = product(cfg->slices, false, true);
        rc = rg_gemm_fp32_ws(xg, w, z, rows, V, D, &g, base + s.gemm, s.gemm_bytes, st, nullptr);
        if (rc != hipSuccess) return rc;
        hipLaunchKernelGGL(loss_parts, dim3((s.parts + 15) / 16, rows), dim3(256), 0, st, z, V, s.parts, part);
        hipLaunchKernelGGL(loss_tokens, dim3((rows + 3) / 4), dim3(256), 0, st, z, V, s.parts, part, first, rows, t,
                           factors, cfg->reduction == RG_LOSS_MEAN ? 1 : 0, tokens, losses);
        if (dx || dw)
            hipLaunchKernelGGL(loss_gradient, dim3((V + 1023) / 1024, rows), dim3(256), 0, st, z, V, first, tokens, t.word);
        if (dx) {
            g = product(cfg->slices, false, false);
            rc = rg_gemm_fp32_ws(z, w, dx + (size_t)first * D, rows, D, V, &g, base + s.gemm, s.gemm_bytes, st, nullptr);
            if (rc != hipSuccess) return rc;
        }
        if (dw) {
            g = product(cfg->slices, true, false);
            rc = rg_gemm_fp32_ws(z, xg, first == 0 ? dw : more, V, D, rows, &g, base + s.gemm, s.gemm_bytes, st, nullptr);
            if (rc != hipSuccess) return rc;
            const size_t n = (size_t)V * D;
            if (first > 0) hipLaunchKernelGGL(loss_add, dim3(grid_of(n)), dim3(256), 0, st, dw, more, n);
        }
    }
    if (dx) hipLaunchKernelGGL(loss_target_dx, dim3(std::min(N, 1 << 20)), dim3(256), 0, st, dx, w, D, tokens, t.word, N);
    if (dw) hipLaunchKernelGGL(loss_target_dw, dim3(N), dim3(256), 0, st, dw, x, D, tokens, t, N);
    if (loss && cfg->reduction == RG_LOSS_NONE) {
        rc = hipMemcpyAsync(loss, losses, (size_t)N * sizeof(float), hipMemcpyDeviceToDevice, st);
        if (rc != hipSuccess) return rc;
    } else if (loss) {
        rg_sum_config sc;
        rg_sum_config_init(&sc);
        rc = rg_sum_fp32_ws(losses, loss, 1, 1, N, &sc, base + s.sum, s.sum_bytes, st);
        if (rc != hipSuccess) return rc;
        if (cfg->reduction == RG_LOSS_MEAN) hipLaunchKernelGGL(loss_mean, dim3(1), dim3(1), 0, st, loss, t.used);
    }
    return hipGetLastError();
}

int rg_scale_fp32(float* x, const float* factor, size_t n, void* stream) {
    if (n == 0) return hipSuccess;
    if (!x || !factor) return hipErrorInvalidValue;
    const unsigned grid = (unsigned)std::min<size_t>((n + 1023) / 1024, 8192);
    hipLaunchKernelGGL(rg::scale_kernel, dim3(grid), dim3(256), 0, static_cast<hipStream_t>(stream), x, factor, n);
    return hipGetLastError();
}

}  // extern "C"
