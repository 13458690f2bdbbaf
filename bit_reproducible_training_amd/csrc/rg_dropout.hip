// Dropout whose random bits come from a counter, so that no mask is stored: a thread makes the four words of four
// consecutive values.
//
// HBM bounds it at 8 bytes a value: 32768 x 2048 in 88 us, 6.1 TB/s, where the generator alone would take 20 (a call of four words
// 214 cycles a wavefront and SIMD).
#include "rg_internal.h"
#include "repro_dropout.h"
#include "repro_dropout_math.h"

namespace rg {
namespace {

constexpr int MAX_BLOCKS = 1 << 16;

// ALIGNED: x and y at multiples of 16 bytes.
template <bool ALIGNED>
__global__ void __launch_bounds__(256)
dropout(const float* x, float* y, size_t n, uint32_t threshold, float factor, uint64_t seed,
        const unsigned long long* seed_at, unsigned long long* used) {
    if (seed_at) seed = *seed_at;
    if (used && blockIdx.x == 0 && threadIdx.x == 0) *used = seed;
    const size_t groups = (n + 3) / 4;
    for (size_t g = (size_t)blockIdx.x * 256 + threadIdx.x; g < groups; g += (size_t)gridDim.x * 256) {
        const size_t at = 4 * g;
        float v[4];
        if (ALIGNED && at + 4 <= n) {
            const float4 f = *reinterpret_cast<const float4*>(x + at);
            v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        } else {
            for (int i = 0; i < 4; ++i) v[i] = at + i < n ? x[at + i] : 0.0f;
        }
        const repro_dropout::Words w = repro_dropout::value_words(g, seed);
        for (int i = 0; i < 4; ++i) v[i] = w.w[i] >= threshold ? v[i] * factor : 0.0f;
        if (ALIGNED && at + 4 <= n) {
            *reinterpret_cast<float4*>(y + at) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            for (int i = 0; i < 4; ++i)
                if (at + i < n) y[at + i] = v[i];
        }
    }
}

}  // namespace
}  // namespace rg

extern "C" int rg_dropout_fp32(const float* x, float* y, size_t n, double p, unsigned long long seed,
                               const unsigned long long* seed_at, unsigned long long* used, void* stream) {
    const auto off = [](const void* a, uintptr_t to) { return (reinterpret_cast<uintptr_t>(a) & (to - 1)) != 0; };
    if (!(p >= 0.0 && p < 1.0) || (n > 0 && (!x || !y)) || off(x, 4) || off(y, 4) || off(seed_at, 8) || off(used, 8))
        return hipErrorInvalidValue;
    if (n == 0 && !used) return hipSuccess;
    const size_t blocks = ((n + 3) / 4 + 255) / 256;
    const dim3 grid((unsigned)(blocks < 1 ? 1 : blocks < rg::MAX_BLOCKS ? blocks : rg::MAX_BLOCKS));
    auto kernel = off(x, 16) || off(y, 16) ? rg::dropout<false> : rg::dropout<true>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), x, y, n,
                       repro_dropout::threshold_of(p), repro_dropout::factor_of(p), seed, seed_at, used);
    return hipGetLastError();
}
