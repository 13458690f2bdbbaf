// Attention over states of another or the same length: the entries and the small kernels.
#include "rg_attention.h"

#include <cmath>
#include <initializer_list>

namespace rg {
namespace attention {

// The mask's truth values as words of 64 keys.
__global__ void __launch_bounds__(256)
pack_mask(const unsigned char* mask, long long heads, long long queries, long long Tk, long long s0, long long s1, long long s2,
          long long key_stride, long long count, unsigned long long* words) {
    const long long W = (Tk + 63) / 64;
    for (long long n = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); n < count; n += (long long)gridDim.x * 4) {
        const long long row = n / W, w = n % W, i = row % queries, h = row / queries % heads, b = row / queries / heads;
        const long long j = 64 * w + (threadIdx.x & 63);
        const bool seen = j < Tk && mask[b * s0 + h * s1 + i * s2 + j * key_stride] != 0;
        const unsigned long long bits = __ballot(seen);
        if ((threadIdx.x & 63) == 0) words[n] = bits;
    }
}

// delta = sum over d of dy y, for each row [B][H][Tq]: 16 lanes take a row, four values (and the four 64 on) each, and add what the
// definition adds: values 32, 16, 8 and 4 apart are 8, 4, 2 and 1 lanes apart, and a lane holds the last four.
template <int APART>
__device__ __forceinline__ float turned(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + APART, 0xF, 0xF, true));
}
template <bool QUADS>
__global__ void __launch_bounds__(256)
row_deltas(Problem z, const float* dy, const float* y, float* delta) {
    const int d = 4 * (threadIdx.x & 15);
    const long long rows = (long long)z.B * z.H * z.Tq;
    for (long long n = (long long)blockIdx.x * 16 + (threadIdx.x >> 4); n < (rows + 15) / 16 * 16; n += (long long)gridDim.x * 16) {
        const long long row = n < rows ? n : rows - 1;
        const int i = (int)(row % z.Tq), t = (int)(row / z.Tq), b = t / z.H, h = t % z.H;
        const size_t at = (((size_t)b * z.Tq + i) * z.H + h) * z.D;
        float s[4] = {};
        const auto take = [&](int from, auto add) {
            float a[4] = {}, c[4] = {};
            if (QUADS) {
                if (from < z.D) {
                    const float4 x = *reinterpret_cast<const float4*>(dy + at + from), w = *reinterpret_cast<const float4*>(y + at + from);
                    a[0] = x.x, a[1] = x.y, a[2] = x.z, a[3] = x.w;
                    c[0] = w.x, c[1] = w.y, c[2] = w.z, c[3] = w.w;
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (from + k < z.D) a[k] = dy[at + from + k], c[k] = y[at + from + k];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (from + k < z.D) s[k] = decltype(add)::value ? __builtin_fmaf(a[k], c[k], s[k]) : a[k] * c[k];
        };
        take(d, std::false_type());
        if (z.D > 64) take(d + 64, std::true_type());
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            s[k] = s[k] + turned<8>(s[k]);
            s[k] = s[k] + turned<4>(s[k]);
            s[k] = s[k] + turned<2>(s[k]);
            s[k] = s[k] + turned<1>(s[k]);
        }
        const float sum = (s[0] + s[2]) + (s[1] + s[3]);
        if (d == 0 && n < rows) delta[n] = sum;
    }
}

__global__ void __launch_bounds__(256)
clear(float* p, size_t n) {
    for (size_t at = (size_t)blockIdx.x * 256 + threadIdx.x; at < n; at += (size_t)gridDim.x * 256) p[at] = 0.0f;
}

namespace {

bool off(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

bool sizes_ok(const rg_attention_config* c) {
    if (!c || c->B < 0 || c->Tq < 0 || c->Tk < 0 || c->H < 1 || c->KVH < 1 || c->H % c->KVH != 0 || c->D < 1 ||
        c->D > RG_ATTENTION_MAX_D || c->Tq > RG_ATTENTION_MAX_LENGTH || c->Tk > RG_ATTENTION_MAX_LENGTH ||
        c->B > RG_ATTENTION_MAX_HEADS || c->B * c->H > RG_ATTENTION_MAX_HEADS || !std::isfinite(c->scale) ||
        !std::isfinite((float)(c->scale * 1.4426950408889634)) || !(c->dropout >= 0.0 && c->dropout < 1.0))
        return false;
    for (int n = 0; n < 3; ++n)
        if (c->q_stride[n] < 0 || c->k_stride[n] < 0 || c->v_stride[n] < 0 || c->mask_stride[n] < 0) return false;
    return c->q_stride[1] <= MAX_ROW && c->k_stride[1] <= MAX_ROW && c->v_stride[1] <= MAX_ROW && (long long)c->H * c->D <= MAX_ROW;
}

Problem problem_of(const rg_attention_config* c, const float* q, const float* k, const float* v, const long long* key_lengths,
                   const unsigned long long* mask, const float* bias, const unsigned long long* seed_at,
                   std::initializer_list<const float*> dense = {}) {
    Problem z;
    z.q = q, z.k = k, z.v = v, z.key_lengths = key_lengths, z.mask = mask, z.bias = bias, z.seed_at = seed_at;
    z.seed = c->seed;
    z.B = (int)c->B, z.Tq = (int)c->Tq, z.Tk = (int)c->Tk, z.H = c->H, z.KVH = c->KVH, z.D = c->D, z.group = c->H / c->KVH;
    // past the ends, the queries all see every key or none
    const long long s = c->query_start;
    z.causal = c->causal && s < c->Tk;
    z.start = (int)(s > c->Tk ? c->Tk : s < -c->Tq ? -c->Tq : s);
    z.factor = std::fabs(repro_attention::score_factor(c->scale));
    z.flip = c->scale < 0.0;
    z.scale = (float)c->scale;
    z.keep_factor = repro_dropout::factor_of(c->dropout);
    z.threshold = repro_dropout::threshold_of(c->dropout);
    uintptr_t odd = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
    for (const float* p : dense) odd |= reinterpret_cast<uintptr_t>(p);
    for (int n = 0; n < 3; ++n) odd |= (uintptr_t)(c->q_stride[n] | c->k_stride[n] | c->v_stride[n]) * sizeof(float);
    z.quads = (odd & 15) == 0 && c->D % 4 == 0;
    for (int n = 0; n < 3; ++n) {
        z.q_stride[n] = c->q_stride[n];
        z.k_stride[n] = c->k_stride[n];
        z.v_stride[n] = c->v_stride[n];
        z.mask_stride[n] = c->mask_stride[n];
    }
    // of a single row the stride says nothing
    if (c->Tq <= 1) z.q_stride[1] = z.D;
    if (c->Tk <= 1) z.k_stride[1] = z.v_stride[1] = z.D;
    z.overlap = z.q_stride[1] < z.D || z.k_stride[1] < z.D || z.v_stride[1] < z.D;
    return z;
}

bool operands_ok(const rg_attention_config* c, const float* q, const float* k, const float* v, const long long* key_lengths,
                 const unsigned long long* mask, const float* bias, const unsigned long long* seed_at) {
    const bool rows = c->B > 0 && c->Tq > 0, keys = c->B > 0 && c->Tk > 0;
    return !(rows && !q) && !(keys && (!k || !v)) && !off(q, 4) && !off(k, 4) && !off(v, 4) && !off(key_lengths, 8) &&
           !off(mask, 8) && !off(bias, 4) && !off(seed_at, 8);
}

}  // namespace
}  // namespace attention
}  // namespace rg

extern "C" {

void rg_attention_config_init(rg_attention_config* cfg) {
    if (!cfg) return;
    *cfg = rg_attention_config{};
    cfg->B = 1;
    cfg->H = cfg->KVH = 1;
    cfg->scale = 1.0;
}

int rg_attention_pack_mask(const unsigned char* mask, long long items, long long heads, long long queries, long long Tk,
                           const long long stride[3], long long key_stride, unsigned long long* words, void* stream) {
    using namespace rg::attention;
    if (items < 0 || heads < 0 || queries < 0 || Tk < 0 || items > RG_ATTENTION_MAX_HEADS || heads > RG_ATTENTION_MAX_HEADS ||
        queries > RG_ATTENTION_MAX_LENGTH || Tk > RG_ATTENTION_MAX_LENGTH || off(words, 8))
        return hipErrorInvalidValue;
    const long long rows = items * heads * queries, W = (Tk + 63) / 64;
    if (rows == 0 || W == 0) return hipSuccess;
    if (!mask || !words || !stride) return hipErrorInvalidValue;
    hipLaunchKernelGGL(pack_mask, dim3(grid_of(rows * W, 4)), dim3(256), 0, static_cast<hipStream_t>(stream), mask, heads,
                       queries, Tk, stride[0], stride[1], stride[2], key_stride, rows * W, words);
    return hipGetLastError();
}

int rg_attention_workspace(const rg_attention_config* cfg, int masked, size_t* bytes) {
    using namespace rg::attention;
    if (!sizes_ok(cfg) || !bytes) return hipErrorInvalidValue;
    *bytes = forward_workspace(problem_of(cfg, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr), masked != 0);
    return hipSuccess;
}

int rg_attention_fp32(const rg_attention_config* cfg, const float* q, const float* k, const float* v,
                      const long long* key_lengths, const unsigned long long* mask, const float* relative_bias,
                      const unsigned long long* seed_at, unsigned long long* used, float* y, float* stats, void* workspace,
                      size_t workspace_bytes, void* stream) {
    using namespace rg::attention;
    if (!sizes_ok(cfg) || !operands_ok(cfg, q, k, v, key_lengths, mask, relative_bias, seed_at) || off(y, 4) ||
        off(stats, 8) || off(used, 8))
        return hipErrorInvalidValue;
    const long long rows = cfg->B * cfg->H * cfg->Tq;
    if (rows > 0 && !y) return hipErrorInvalidValue;
    if (rows == 0) return hipSuccess;
    const Problem z = problem_of(cfg, q, k, v, key_lengths, mask, relative_bias, seed_at, {y});
    const size_t needed = forward_workspace(z, mask != nullptr);
    if (needed > 0 && (!workspace || workspace_bytes < needed || off(workspace, 16))) return hipErrorInvalidValue;
    return forward(z, y, stats, used, workspace, static_cast<hipStream_t>(stream));
}

int rg_attention_grad_workspace(const rg_attention_config* cfg, int want_bias, size_t* bytes) {
    using namespace rg::attention;
    if (!sizes_ok(cfg) || !bytes) return hipErrorInvalidValue;
    const Problem z = problem_of(cfg, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
    *bytes = z.B > 0 && z.Tq > 0 && z.Tk > 0 ? backward_workspace(z, want_bias != 0) : 0;
    return hipSuccess;
}

int rg_attention_grad_fp32(const rg_attention_config* cfg, const float* dy, const float* q, const float* k, const float* v,
                           const long long* key_lengths, const unsigned long long* mask, const float* relative_bias,
                           const unsigned long long* seed_at, const float* y, const float* stats, float* dq, float* dk,
                           float* dv, float* drelative_bias, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace rg::attention;
    if (!sizes_ok(cfg) || !operands_ok(cfg, q, k, v, key_lengths, mask, relative_bias, seed_at) || off(dy, 4) || off(y, 4) ||
        off(stats, 8) || off(dq, 4) || off(dk, 4) || off(dv, 4) || off(drelative_bias, 4) || (drelative_bias && !relative_bias))
        return hipErrorInvalidValue;
    const long long rows = cfg->B * cfg->H * cfg->Tq, keys = cfg->B * cfg->KVH * cfg->Tk;
    size_t needed = 0;
    (void)rg_attention_grad_workspace(cfg, drelative_bias != nullptr, &needed);
    if ((rows > 0 && (!dy || !y || !stats || !dq)) || (keys > 0 && (!dk || !dv)) ||
        (needed > 0 && (!workspace || workspace_bytes < needed || off(workspace, 16))))
        return hipErrorInvalidValue;
    const Problem z = problem_of(cfg, q, k, v, key_lengths, mask, relative_bias, seed_at, {dy, dk, dv});
    hipStream_t st = static_cast<hipStream_t>(stream);
    const long long columns = drelative_bias ? (long long)z.H * (z.Tq + z.Tk - 1) : 0;
    if (rows == 0 || keys == 0) {  // no pair: zeros
        const auto zero = [&](float* p, long long n) {
            if (p && n > 0) hipLaunchKernelGGL(clear, dim3(grid_of(n, 256)), dim3(256), 0, st, p, (size_t)n);
        };
        zero(dq, rows * z.D);
        zero(dk, keys * z.D);
        zero(dv, keys * z.D);
        zero(drelative_bias, columns);
        return hipGetLastError();
    }
    const bool quads = z.D % 4 == 0 && !off(dy, 16) && !off(y, 16);
    hipLaunchKernelGGL(quads ? row_deltas<true> : row_deltas<false>, dim3(grid_of(rows, 16)), dim3(256), 0, st, z, dy, y,
                       static_cast<float*>(workspace));
    return backward(z, dy, stats, dq, dk, dv, drelative_bias, workspace, st);
}

}  // extern "C"
