// The AdamW step over a list of tensors, with the moments in float32 or in 8 bits.
//
// A launch takes up to a fixed number of tensors in its arguments (no table in device memory to
// copy there first), and its blocks are dealt to them by chunks: a block finds its tensor by the
// tensors' first chunks, all read at once.
//
// In float32 HBM bounds it: 28 bytes a value, 640 us for 124 million values of 148 tensors, 5.4 TB/s where a
// copy of 1 GiB reaches 5.1. With moments in 8 bits 16 bytes a value remain and the vector units bound it, see there.
#include "rg_internal.h"
#include "repro_adamw.h"
#include "repro_adamw_math.h"

#include <cmath>
#include <cstdint>

namespace rg {
namespace {

using repro_adamw::BLOCK;
using repro_adamw::Scalars;

static_assert(BLOCK == RG_ADAMW8_BLOCK && BLOCK == 4 * 64, "a wavefront holds a block, four values a lane");

constexpr int THREADS = 256;
constexpr long long MOST = 1ll << 30;  // values of one entry: a longer tensor takes several

struct Entry {
    float* p;
    const float* g;
    float* m;
    float* v;
    uint32_t n;  // values
};
struct Entry8 {
    float* p;
    const float* g;
    uint8_t *m, *m_exp, *v, *v_exp;
    uint32_t n;
    uint32_t block;  // the call's blocks before this entry
};
// Where all tensors' moments lie one after another, from the call's first block on (adamw8_state makes them so; the
// optimizer keeps each parameter's by itself), an entry needs no addresses of its own for them, and a launch takes 128 tensors instead of 66: a step of 300
// small tensors 29 us by five launches, 18 by three.
struct EntryInRow {
    float* p;
    const float* g;
    uint32_t n;
    uint32_t block;
};
template <class E>
struct Shared {};
template <>
struct Shared<EntryInRow> {
    uint8_t *m, *m_exp, *v, *v_exp;
};
// As many as the 4 KiB of a launch's arguments hold, two a lane at most. first: the entries' first chunks in
// this launch, past the last entry a number that no chunk has.
template <class E>
struct List {
    static constexpr size_t FIT = (4096 - 96) / (sizeof(E) + 4);
    static constexpr int MAX = FIT < 128 ? FIT : 128;
    Scalars s;
    Shared<E> shared;
    uint32_t first[MAX];
    E e[MAX];
};
static_assert(List<Entry>::MAX == 90 && List<Entry8>::MAX == 66 && List<EntryInRow>::MAX == 128, "tensors a launch");
static_assert(sizeof(List<Entry>) <= 4096 && sizeof(List<Entry8>) <= 4096 && sizeof(List<EntryInRow>) <= 4096,
              "launch arguments");

__device__ __forceinline__ Entry8 entry8(const List<Entry8>& list, int i) { return list.e[i]; }
__device__ __forceinline__ Entry8 entry8(const List<EntryInRow>& list, int i) {
    const EntryInRow& e = list.e[i];
    const Shared<EntryInRow>& t = list.shared;
    const size_t b = e.block, at = b * BLOCK;
    return Entry8{e.p, e.g, t.m + at, t.m_exp + b, t.v + at, t.v_exp + b, e.n, e.block};
}

// The entry of a chunk: the lanes read every entry's first chunk at once, where a bisection reads six in
// turn (launch arguments are far from the GPU: small tensors' launches took 7.1 us, of 4.5 so).
template <class E>
__device__ __forceinline__ int entry_of(const List<E>& list, uint32_t chunk) {
    const int lane = threadIdx.x & 63;
    uint32_t a = lane < List<E>::MAX ? list.first[lane] : ~0u;
    uint32_t b = lane + 64 < List<E>::MAX ? list.first[lane + 64] : ~0u;
    return __popcll(__ballot(a <= chunk)) + __popcll(__ballot(b <= chunk)) - 1;
}

// What a step reads is written again or not needed any more: its loads leave nothing in the caches (124 million values 658
// -> 640 us; with the moments' stores past the caches too 642. In the 8-bit step 435 -> 423, but reading the moments back
// right after it took 10 longer).
typedef float v4f __attribute__((ext_vector_type(4)));
__device__ __forceinline__ v4f load_once(const float* p) { return __builtin_nontemporal_load(reinterpret_cast<const v4f*>(p)); }

// A chunk is 4 U values a thread. 16-byte accesses where all four arrays allow them, else single
// values, neighbouring threads on neighbouring values either way.
template <int U>
__global__ void __launch_bounds__(THREADS)
adamw_kernel(const List<Entry> list) {
    const int entry = entry_of(list, blockIdx.x);
    const Entry& t = list.e[entry];
    const Scalars s = list.s;
    const uint32_t base = (blockIdx.x - list.first[entry]) * (uint32_t)(THREADS * 4 * U);
    const uint32_t left = t.n - base;
    float* __restrict__ p = t.p + base;
    const float* __restrict__ g = t.g + base;
    float* __restrict__ m = t.m + base;
    float* __restrict__ v = t.v + base;
    const uintptr_t off = reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g) |
                          reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v);
    if ((off & 15) == 0 && left >= (uint32_t)(THREADS * 4 * U)) {
        v4f pv[U], gv[U], mv[U], vv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t i = u * THREADS + threadIdx.x;
            pv[u] = load_once(p + 4 * i);
            gv[u] = load_once(g + 4 * i);
            mv[u] = load_once(m + 4 * i);
            vv[u] = load_once(v + 4 * i);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t i = u * THREADS + threadIdx.x;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float mk = mv[u][k], vk = vv[u][k];
                pv[u][k] = repro_adamw::update(pv[u][k], gv[u][k], mk, vk, s);
                mv[u][k] = mk;
                vv[u][k] = vk;
            }
            reinterpret_cast<v4f*>(p)[i] = pv[u];
            reinterpret_cast<v4f*>(m)[i] = mv[u];
            reinterpret_cast<v4f*>(v)[i] = vv[u];
        }
        return;
    }
    const uint32_t n = left < (uint32_t)(THREADS * 4 * U) ? left : (uint32_t)(THREADS * 4 * U);
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
        float mi = m[i], vi = v[i];
        p[i] = repro_adamw::update(p[i], g[i], mi, vi, s);
        m[i] = mi;
        v[i] = vi;
    }
}

template <int CTRL>
__device__ __forceinline__ uint32_t rotated(uint32_t a) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, CTRL, 0xF, 0xF, true);
}
// The largest over the wavefront, as a scalar: half waves, rows of 16, and rotations inside a row.
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t a) {
    auto s = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    a = max((uint32_t)s[0], (uint32_t)s[1]);
    s = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    a = max((uint32_t)s[0], (uint32_t)s[1]);
    a = max(a, rotated<0x128>(a));
    a = max(a, rotated<0x124>(a));
    a = max(a, rotated<0x122>(a));
    a = max(a, rotated<0x121>(a));
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)a);
}

// One block of BLOCK values by a wavefront, its lane l the values 4 l .. 4 l + 3. FULL: the tensor holds the
// whole block and 16-byte accesses are allowed.
template <bool FULL>
struct Block8 {
    float p[4], g[4];
    uint32_t m, v;  // codes
    int me, ve;

    __device__ __forceinline__ void load(const Entry8& t, uint32_t b, int lane) {
        const uint32_t at = b * BLOCK + 4 * lane;
        m = reinterpret_cast<const uint32_t*>(t.m + (size_t)b * BLOCK)[lane];
        v = reinterpret_cast<const uint32_t*>(t.v + (size_t)b * BLOCK)[lane];
        me = t.m_exp[b];
        ve = t.v_exp[b];
        if constexpr (FULL) {
            const float4 pp = *reinterpret_cast<const float4*>(t.p + at), gg = *reinterpret_cast<const float4*>(t.g + at);
            p[0] = pp.x, p[1] = pp.y, p[2] = pp.z, p[3] = pp.w;
            g[0] = gg.x, g[1] = gg.y, g[2] = gg.z, g[3] = gg.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[i] = at + i < t.n ? t.p[at + i] : 0.0f;
                g[i] = at + i < t.n ? t.g[at + i] : 0.0f;
            }
        }
    }
    __device__ __forceinline__ void step(const Entry8& t, uint32_t b, int lane, const Scalars& s) {
        const uint32_t at = b * BLOCK + 4 * lane;
        const int em0 = __builtin_amdgcn_readfirstlane(me), ev0 = __builtin_amdgcn_readfirstlane(ve);
        float mv[4], vv[4];
        uint32_t top_m = 0, top_v = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            mv[i] = repro_adamw::decode_m((uint8_t)(m >> (8 * i)), em0);
            vv[i] = repro_adamw::decode_v((uint8_t)(v >> (8 * i)), ev0);
            p[i] = repro_adamw::update(p[i], g[i], mv[i], vv[i], s);
            if (!FULL && at + i >= t.n) mv[i] = vv[i] = 0.0f;  // past the tensor: codes of zero
            top_m = max(top_m, repro_adamw::magnitude_bits(mv[i]));
            top_v = max(top_v, repro_adamw::magnitude_bits(vv[i]));
        }
        const int em = repro_adamw::shared_exponent(wave_max_bits(top_m), repro_adamw::SPAN_M);
        const int ev = repro_adamw::shared_exponent(wave_max_bits(top_v), repro_adamw::SPAN_V);
        uint32_t cm = 0, cv = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = repro_adamw::rounding((t.block + b) * BLOCK + 4 * lane + i, s.salt);
            cm |= (uint32_t)repro_adamw::encode_m(mv[i], em, u & 0xFFFFu) << (8 * i);
            cv |= (uint32_t)repro_adamw::encode_v(vv[i], ev, u >> 16) << (8 * i);
        }
        reinterpret_cast<uint32_t*>(t.m + (size_t)b * BLOCK)[lane] = cm;
        reinterpret_cast<uint32_t*>(t.v + (size_t)b * BLOCK)[lane] = cv;
        if (lane == 0) {
            t.m_exp[b] = (uint8_t)em;
            t.v_exp[b] = (uint8_t)ev;
        }
        if constexpr (FULL) {
            *reinterpret_cast<float4*>(t.p + at) = make_float4(p[0], p[1], p[2], p[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (at + i < t.n) t.p[at + i] = p[i];
        }
    }
};

// A wavefront takes U blocks in turn, all of them loaded before the first is stepped. (Eight a wavefront in a loop,
// fewer searches of the list: no faster. The arithmetic bounds it: about 100 vector instructions a
// value, 430 to 465 us for 124 million of them.)
template <int U, class E>
__global__ void __launch_bounds__(THREADS)
adamw8_kernel(const List<E> list) {
    const int entry = entry_of(list, blockIdx.x);
    const Entry8 t = entry8(list, entry);
    const Scalars s = list.s;
    const int lane = threadIdx.x & 63;
    const uint32_t blocks = (t.n + BLOCK - 1) / BLOCK;
    const uint32_t b0 = (blockIdx.x - list.first[entry]) * (uint32_t)(THREADS / 64 * U) +
                        (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool wide = ((reinterpret_cast<uintptr_t>(t.p) | reinterpret_cast<uintptr_t>(t.g)) & 15) == 0;
    if (wide && b0 + (U - 1) * (THREADS / 64) < t.n / BLOCK) {
        Block8<true> k[U];
#pragma unroll
        for (int u = 0; u < U; ++u) k[u].load(t, b0 + u * (THREADS / 64), lane);
#pragma unroll
        for (int u = 0; u < U; ++u) k[u].step(t, b0 + u * (THREADS / 64), lane, s);
        return;
    }
    for (uint32_t b = b0; b < blocks && b < b0 + U * (THREADS / 64); b += THREADS / 64) {
        Block8<false> k;
        k.load(t, b, lane);
        k.step(t, b, lane, s);
    }
}

__global__ void __launch_bounds__(THREADS)
adamw8_values_kernel(const uint8_t* __restrict__ m, const uint8_t* __restrict__ m_exp,
                     const uint8_t* __restrict__ v, const uint8_t* __restrict__ v_exp,
                     float* __restrict__ m_values, float* __restrict__ v_values, long long blocks) {
    const int lane = threadIdx.x & 63;
    for (long long b = (long long)blockIdx.x * (THREADS / 64) + (threadIdx.x >> 6); b < blocks;
         b += (long long)gridDim.x * (THREADS / 64)) {
        const uint32_t mc = reinterpret_cast<const uint32_t*>(m + b * BLOCK)[lane];
        const uint32_t vc = reinterpret_cast<const uint32_t*>(v + b * BLOCK)[lane];
        const int me = m_exp[b], ve = v_exp[b];
        float mo[4], vo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            mo[i] = repro_adamw::decode_m((uint8_t)(mc >> (8 * i)), me);
            vo[i] = repro_adamw::decode_v((uint8_t)(vc >> (8 * i)), ve);
        }
        reinterpret_cast<float4*>(m_values + b * BLOCK)[lane] = make_float4(mo[0], mo[1], mo[2], mo[3]);
        reinterpret_cast<float4*>(v_values + b * BLOCK)[lane] = make_float4(vo[0], vo[1], vo[2], vo[3]);
    }
}

bool config_ok(const rg_adamw_config* c) {
    return c != nullptr && c->lr >= 0.0 && c->eps >= 0.0 && c->weight_decay >= 0.0 && c->beta1 >= 0.0 &&
           c->beta1 < 1.0 && c->beta2 >= 0.0 && c->beta2 < 1.0 && c->step >= 1;
}

bool off(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

// Fills lists of entries and launches each as it is full.
template <class E, class Launch>
struct Dealer {
    List<E> list;
    int count = 0;
    uint32_t chunks = 0;
    int rc = hipSuccess;
    Launch launch;
    Dealer(const Scalars& s, Launch l) : launch(l) { list.s = s; }
    void flush() {
        if (count == 0 || rc != hipSuccess) return;
        for (int i = count; i < List<E>::MAX; ++i) list.first[i] = ~0u;
        launch(list, chunks);
        rc = hipGetLastError();
        count = 0;
        chunks = 0;
    }
    void add(const E& e, uint32_t n) {
        if (count == List<E>::MAX || (uint64_t)chunks + n > 0xFFFFFFu) flush();  // 2^32 threads
        list.first[count] = chunks;
        list.e[count++] = e;
        chunks += n;
    }
};

template <class E, class Launch>
Dealer<E, Launch> make_dealer(const Scalars& s, Launch l) {
    return Dealer<E, Launch>(s, l);
}

Scalars scalars_of(const rg_adamw_config* c) {
    return repro_adamw::make_scalars(c->lr, c->beta1, c->beta2, c->eps, c->weight_decay, c->step);
}

}  // namespace
}  // namespace rg

extern "C" {

void rg_adamw_config_init(rg_adamw_config* cfg) {
    if (!cfg) return;
    cfg->lr = 1e-3;
    cfg->beta1 = 0.9;
    cfg->beta2 = 0.999;
    cfg->eps = 1e-8;
    cfg->weight_decay = 1e-2;
    cfg->step = 1;
}

int rg_adamw_fp32(const rg_adamw_tensor* tensors, int count, const rg_adamw_config* cfg, void* stream) {
    using namespace rg;
    if (!config_ok(cfg) || count < 0 || (count > 0 && !tensors)) return hipErrorInvalidValue;
    for (int i = 0; i < count; ++i) {
        const rg_adamw_tensor& t = tensors[i];
        if (t.n < 0) return hipErrorInvalidValue;
        if (t.n > 0 && (!t.p || !t.g || !t.m || !t.v || off(t.p, 4) || off(t.g, 4) || off(t.m, 4) || off(t.v, 4)))
            return hipErrorInvalidValue;
    }
    constexpr int U = 4;
    constexpr uint32_t CHUNK = THREADS * 4 * U;
    hipStream_t st = static_cast<hipStream_t>(stream);
    auto dealer = make_dealer<Entry>(scalars_of(cfg), [&](const List<Entry>& list, uint32_t chunks) {
        hipLaunchKernelGGL(adamw_kernel<U>, dim3(chunks), dim3(THREADS), 0, st, list);
    });
    for (int i = 0; i < count; ++i) {
        const rg_adamw_tensor& t = tensors[i];
        for (long long a = 0; a < t.n; a += MOST) {
            Entry e;
            e.p = t.p + a;
            e.g = t.g + a;
            e.m = t.m + a;
            e.v = t.v + a;
            e.n = (uint32_t)(t.n - a < MOST ? t.n - a : MOST);
            dealer.add(e, (e.n + CHUNK - 1) / CHUNK);
        }
    }
    dealer.flush();
    return dealer.rc;
}

int rg_adamw8_fp32(const rg_adamw8_tensor* tensors, int count, const rg_adamw_config* cfg, void* stream) {
    using namespace rg;
    if (!config_ok(cfg) || count < 0 || (count > 0 && !tensors)) return hipErrorInvalidValue;
    for (int i = 0; i < count; ++i) {
        const rg_adamw8_tensor& t = tensors[i];
        if (t.n < 0) return hipErrorInvalidValue;
        if (t.n > 0 && (!t.p || !t.g || !t.m || !t.m_exp || !t.v || !t.v_exp || off(t.p, 4) || off(t.g, 4) ||
                        off(t.m, 4) || off(t.v, 4)))
            return hipErrorInvalidValue;
    }
    bool in_row = true;
    const rg_adamw8_tensor* start = nullptr;
    long long before = 0;
    for (int i = 0; i < count; ++i) {
        const rg_adamw8_tensor& t = tensors[i];
        if (t.n == 0) continue;
        if (!start) start = &t;
        const long long at = before * BLOCK;
        in_row = in_row && t.m == start->m + at && t.v == start->v + at && t.m_exp == start->m_exp + before &&
                 t.v_exp == start->v_exp + before;
        before += (t.n + BLOCK - 1) / BLOCK;
    }
    constexpr int U = 2;
    constexpr uint32_t CHUNK = THREADS / 64 * U;  // blocks
    hipStream_t st = static_cast<hipStream_t>(stream);
    const auto step = [&](auto dealer, auto entry) {
        uint32_t block = 0;
        for (int i = 0; i < count; ++i) {
            const rg_adamw8_tensor& t = tensors[i];
            for (long long a = 0; a < t.n; a += MOST) {
                const uint32_t n = (uint32_t)(t.n - a < MOST ? t.n - a : MOST), blocks = (n + BLOCK - 1) / BLOCK;
                dealer.add(entry(t, a, n, block), (blocks + CHUNK - 1) / CHUNK);
                block += blocks;
            }
        }
        dealer.flush();
        return dealer.rc;
    };
    if (in_row && start) {
        auto dealer = make_dealer<EntryInRow>(scalars_of(cfg), [&](const List<EntryInRow>& list, uint32_t chunks) {
            hipLaunchKernelGGL((adamw8_kernel<U, EntryInRow>), dim3(chunks), dim3(THREADS), 0, st, list);
        });
        dealer.list.shared = Shared<EntryInRow>{start->m, start->m_exp, start->v, start->v_exp};
        return step(dealer, [](const rg_adamw8_tensor& t, long long a, uint32_t n, uint32_t block) {
            return EntryInRow{t.p + a, t.g + a, n, block};
        });
    }
    return step(make_dealer<Entry8>(scalars_of(cfg), [&](const List<Entry8>& list, uint32_t chunks) {
        hipLaunchKernelGGL((adamw8_kernel<U, Entry8>), dim3(chunks), dim3(THREADS), 0, st, list);
    }), [](const rg_adamw8_tensor& t, long long a, uint32_t n, uint32_t block) {
        return Entry8{t.p + a, t.g + a, t.m + a, t.m_exp + a / BLOCK, t.v + a, t.v_exp + a / BLOCK, n, block};
    });
}

int rg_adamw8_values(const unsigned char* m, const unsigned char* m_exp, const unsigned char* v,
                     const unsigned char* v_exp, float* m_values, float* v_values, long long blocks,
                     void* stream) {
    using namespace rg;
    if (blocks < 0 || blocks > 2147483647ll) return hipErrorInvalidValue;
    if (blocks == 0) return hipSuccess;
    if (!m || !m_exp || !v || !v_exp || !m_values || !v_values || off(m, 4) || off(v, 4) || off(m_values, 16) ||
        off(v_values, 16))
        return hipErrorInvalidValue;
    const long long needed = (blocks + THREADS / 64 - 1) / (THREADS / 64);
    const unsigned grid = (unsigned)(needed < (1 << 22) ? needed : (1 << 22));
    hipLaunchKernelGGL(adamw8_values_kernel, dim3(grid), dim3(THREADS), 0, static_cast<hipStream_t>(stream), m,
                       m_exp, v, v_exp, m_values, v_values, blocks);
    return hipGetLastError();
}

}  // extern "C"
