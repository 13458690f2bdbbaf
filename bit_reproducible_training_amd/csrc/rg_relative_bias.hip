// The learned bias of relative positions: a table's row for each bucket of distances, laid out by distance or for every
// pair of query and key, and the table's gradient.
//
// A bias depends on the distance alone, so a dense one is written from LDS at the speed of its stores, and a dense
// gradient is first added up along its diagonals, a thread each. 12 x 1024 x 1024: 12.5 us forward (4 TB/s), 11.4 to 18.7 for the diagonals
// by where the gradient lies (4.4 to 2.7 TB/s: a row starts 4 bytes off the one before), 5.2 for the buckets.
#include "rg_internal.h"
#include "repro_attention.h"
#include "repro_attention_math.h"

namespace rg {
namespace {

using repro_attention::bucket_of;
using repro_attention::RUN;
using repro_attention::STRANDS;

struct Borders {
    int count, both, at[RG_RELATIVE_BIAS_MAX_BORDERS];
};
struct Sizes {
    int Tq, Tk, H;
    long long start;
};

__global__ void __launch_bounds__(256)
bias_by_distance(Sizes z, Borders borders, const float* table, float* out) {
    __shared__ int at[RG_RELATIVE_BIAS_MAX_BORDERS];
    for (int n = threadIdx.x; n < borders.count; n += 256) at[n] = borders.at[n];
    __syncthreads();
    const long long columns = (long long)z.Tq + z.Tk - 1, count = columns * z.H;
    for (long long n = (long long)blockIdx.x * 256 + threadIdx.x; n < count; n += (long long)gridDim.x * 256) {
        const int h = (int)(n / columns);
        const long long relative = n % columns - (z.Tq - 1) - z.start;
        out[n] = table[(size_t)bucket_of(relative, at, borders.count, borders.both) * z.H + h];
    }
}

constexpr int ROWS = 32, WIDE = 1024;

// A block writes ROWS rows of WIDE keys of a head, four a thread. QUADS: rows are multiples of 16 bytes.
template <bool QUADS>
__global__ void __launch_bounds__(256)
bias_dense(Sizes z, Borders borders, const float* table, float* out) {
    __shared__ int at[RG_RELATIVE_BIAS_MAX_BORDERS];
    __shared__ float value[WIDE + ROWS];
    for (int n = threadIdx.x; n < borders.count; n += 256) at[n] = borders.at[n];
    const int across = (z.Tk + WIDE - 1) / WIDE, down = (z.Tq + ROWS - 1) / ROWS;
    const long long blocks = (long long)across * down * z.H;
    for (long long block = blockIdx.x; block < blocks; block += gridDim.x) {
        const int j0 = (int)(block % across) * WIDE, i0 = (int)(block / across % down) * ROWS, h = (int)(block / across / down);
        __syncthreads();
        for (int n = threadIdx.x; n < WIDE + ROWS - 1; n += 256) {
            const long long relative = (long long)j0 + n - (ROWS - 1) - i0 - z.start;
            value[n] = table[(size_t)bucket_of(relative, at, borders.count, borders.both) * z.H + h];
        }
        __syncthreads();
        const int c = 4 * threadIdx.x, j = j0 + c;
        if (j >= z.Tk) continue;
        const int rows = min(ROWS, z.Tq - i0);
        float* p = out + ((size_t)h * z.Tq + i0) * z.Tk + j;
        for (int i = 0; i < rows; ++i, p += z.Tk) {
            const float* v = value + c + ROWS - 1 - i;
            if (QUADS) {
                *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
                for (int x = 0; x < 4; ++x)
                    if (j + x < z.Tk) p[x] = v[x];
            }
        }
    }
}

// part[h][run][n]: the sum along a diagonal within a run of RUN rows; n is j - (i - 64 run) + RUN - 1.
__global__ void __launch_bounds__(256)
diagonal_sums(Sizes z, const float* dout, float* part) {
    const int width = z.Tk + RUN - 1, across = (width + 255) / 256, runs = (z.Tq + RUN - 1) / RUN;
    const long long blocks = (long long)across * runs * z.H;
    for (long long block = blockIdx.x; block < blocks; block += gridDim.x) {
        const int n = (int)(block % across) * 256 + threadIdx.x, r = (int)(block / across % runs), h = (int)(block / across / runs);
        if (n >= width) continue;
        const int j0 = n - (RUN - 1);  // the key beside the run's first row
        const int first = max(0, -j0), last = min(min(RUN, z.Tq - r * RUN), z.Tk - j0);
        const float* p = dout + ((size_t)h * z.Tq + r * RUN) * z.Tk;
        float s = 0.0f;
#pragma unroll
        for (int i0 = 0; i0 < RUN; i0 += 16) {  // sixteen loads in flight; those of no pair read the run's first value and are left out
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = p[i0 + i >= first && i0 + i < last ? (size_t)(i0 + i) * (z.Tk + 1) + j0 : 0];
#pragma unroll
            for (int i = 0; i < 16; ++i) s = s + (i0 + i >= first && i0 + i < last ? v[i] : 0.0f);
        }
        part[((size_t)h * runs + r) * width + n] = s;
    }
}

// A block adds up a bucket of a head: the columns [low, high) that the borders give it, column n in strand n mod STRANDS.
__global__ void __launch_bounds__(STRANDS)
bucket_sums(Sizes z, Borders borders, int first_block, const float* dout, const float* part, float* dtable) {
    __shared__ float strand[STRANDS];
    const int half = borders.count + 1, block = first_block + blockIdx.x;
    const int bucket = block / z.H, h = block % z.H;
    const bool after = bucket >= half;
    const int c = after ? bucket - half : bucket;
    const long long never = 1ll << 40, near = c == 0 ? 0 : borders.at[c - 1], far = c + 1 == half ? never : borders.at[c];
    // relative positions [from, to)
    const long long from = after ? (near > 1 ? near : 1) : -far + 1, to = after ? far : c == 0 ? (borders.both ? 1 : never) : -near + 1;
    const long long origin = z.start + z.Tq - 1, columns = (long long)z.Tq + z.Tk - 1;
    const long long low = from + origin > 0 ? from + origin : 0, high = to + origin < columns ? to + origin : columns;
    const int width = z.Tk + RUN - 1, runs = (z.Tq + RUN - 1) / RUN;
    float s = 0.0f;
    long long n = low + ((long long)threadIdx.x - low % STRANDS + STRANDS) % STRANDS;
    for (; n < high; n += STRANDS) {
        float v;
        if (part) {
            const int away = (int)(n - (z.Tq - 1));
            const int first = max(0, -away) / RUN, last = min(z.Tq, z.Tk - away);  // rows max(0, -away) .. last
            const int rows = (last + RUN - 1) / RUN - first;  // runs
            const float* p = part + ((size_t)h * runs + first) * width + away + first * RUN + RUN - 1;
            v = 0.0f;
            for (int r0 = 0; r0 < rows; r0 += 16) {
                float x[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = p[(size_t)min(r0 + r, rows - 1) * (width + RUN)];
#pragma unroll
                for (int r = 0; r < 16; ++r) v = v + (r0 + r < rows ? x[r] : 0.0f);
            }
        } else {
            v = dout[h * columns + n];
        }
        s = s + v;
    }
    strand[threadIdx.x] = s;
    for (int step = STRANDS / 2; step > 0; step /= 2) {
        __syncthreads();
        if (threadIdx.x < step) strand[threadIdx.x] = strand[threadIdx.x] + strand[threadIdx.x + step];
    }
    if (threadIdx.x == 0) dtable[(size_t)bucket * z.H + h] = strand[0] + 0.0f;
}

bool sizes_ok(const rg_relative_bias_config* c) {
    if (!c || c->Tq < 0 || c->Tk < 0 || c->Tq > RG_ATTENTION_MAX_LENGTH || c->Tk > RG_ATTENTION_MAX_LENGTH || c->H < 1 ||
        c->H > RG_ATTENTION_MAX_HEADS || c->query_start > (1ll << 32) || c->query_start < -(1ll << 32) || c->count < 1 ||
        c->count > RG_RELATIVE_BIAS_MAX_BORDERS || !c->borders || c->borders[0] < 1)
        return false;
    for (int n = 1; n < c->count; ++n)
        if (c->borders[n] < c->borders[n - 1]) return false;
    return true;
}

Borders borders_of(const rg_relative_bias_config* c) {
    Borders b;
    b.count = c->count;
    b.both = c->both != 0;
    for (int n = 0; n < RG_RELATIVE_BIAS_MAX_BORDERS; ++n) b.at[n] = n < c->count ? c->borders[n] : 0;
    return b;
}

Sizes sizes_of(const rg_relative_bias_config* c) { return Sizes{(int)c->Tq, (int)c->Tk, c->H, c->query_start}; }

long long values_of(const rg_relative_bias_config* c) {
    return c->Tq + c->Tk == 0 ? 0 : (long long)c->H * (c->dense ? c->Tq * c->Tk : c->Tq + c->Tk - 1);
}

unsigned capped(long long blocks) { return (unsigned)(blocks < (1 << 20) ? blocks : 1 << 20); }

}  // namespace
}  // namespace rg

extern "C" {

int rg_relative_bias_fp32(const rg_relative_bias_config* cfg, const float* table, float* out, void* stream) {
    using namespace rg;
    if (!sizes_ok(cfg) || (reinterpret_cast<uintptr_t>(table) & 3) != 0 || (reinterpret_cast<uintptr_t>(out) & 3) != 0)
        return hipErrorInvalidValue;
    const long long values = values_of(cfg);
    if (values == 0) return hipSuccess;
    if (!table || !out) return hipErrorInvalidValue;
    const Sizes z = sizes_of(cfg);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (cfg->dense) {
        const long long blocks = (long long)((z.Tk + WIDE - 1) / WIDE) * ((z.Tq + ROWS - 1) / ROWS) * z.H;
        auto kernel = z.Tk % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0 ? bias_dense<true> : bias_dense<false>;
        hipLaunchKernelGGL(kernel, dim3(capped(blocks)), dim3(256), 0, st, z, borders_of(cfg), table, out);
    } else {
        hipLaunchKernelGGL(bias_by_distance, dim3(capped((values + 255) / 256)), dim3(256), 0, st, z, borders_of(cfg), table, out);
    }
    return hipGetLastError();
}

int rg_relative_bias_grad_workspace(const rg_relative_bias_config* cfg, size_t* bytes) {
    using namespace rg;
    if (!sizes_ok(cfg) || !bytes) return hipErrorInvalidValue;
    *bytes = cfg->dense && values_of(cfg) > 0
                 ? sizeof(float) * cfg->H * (size_t)((cfg->Tq + RUN - 1) / RUN) * (size_t)(cfg->Tk + RUN - 1) : 0;
    return hipSuccess;
}

int rg_relative_bias_grad_fp32(const rg_relative_bias_config* cfg, const float* dout, float* dtable, void* workspace,
                               size_t workspace_bytes, void* stream) {
    using namespace rg;
    if (!sizes_ok(cfg) || !dtable || (reinterpret_cast<uintptr_t>(dtable) & 3) != 0 || (reinterpret_cast<uintptr_t>(dout) & 3) != 0)
        return hipErrorInvalidValue;
    size_t needed = 0;
    (void)rg_relative_bias_grad_workspace(cfg, &needed);
    const long long values = values_of(cfg);
    if ((values > 0 && !dout) || (needed > 0 && (!workspace || workspace_bytes < needed || (reinterpret_cast<uintptr_t>(workspace) & 3) != 0)))
        return hipErrorInvalidValue;
    const int sums = (cfg->count + 1) * (cfg->both ? 2 : 1) * cfg->H, most = 1 << 23;  // (of a launch: it takes fewer than 2^32 threads)
    Sizes z = sizes_of(cfg);
    if (values == 0) z.Tq = 1, z.Tk = 0;  // no column: every sum is 0
    hipStream_t st = static_cast<hipStream_t>(stream);
    float* part = needed > 0 ? static_cast<float*>(workspace) : nullptr;
    if (part) {
        const long long blocks = (long long)((z.Tk + RUN - 1 + 255) / 256) * ((z.Tq + RUN - 1) / RUN) * z.H;
        hipLaunchKernelGGL(diagonal_sums, dim3(capped(blocks)), dim3(256), 0, st, z, dout, part);
    }
    for (int first = 0; first < sums; first += most)
        hipLaunchKernelGGL(bucket_sums, dim3((unsigned)(sums - first < most ? sums - first : most)), dim3(STRANDS), 0, st, z, borders_of(cfg), first,
                           dout, part, dtable);
    return hipGetLastError();
}

}  // extern "C"
