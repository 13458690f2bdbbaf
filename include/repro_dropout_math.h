#pragma once
// What defines the reproducible dropout: its random bits, callable from host and device code. A mask is never
// stored: every pass makes the bits it needs again from a seed and a value's place.
//
// Philox 4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, 2011): ten rounds of two
// 32 x 32 -> 64 bit products turn a counter of four words, under a key of two, into four random words.
#include "repro_gemm_math.h"

namespace repro_dropout {

struct Words {
    uint32_t w[4];
};

RG_HD inline Words philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint64_t seed) {
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return Words{{c0, c1, c2, c3}};
}

// A value is kept where its word is at least this: p 2^32 rounded down, for 0 <= p < 1.
inline uint32_t threshold_of(double p) { return (uint32_t)(p * 4294967296.0); }
// What kept values are multiplied by.
inline float factor_of(double p) { return (float)(1.0 / (1.0 - p)); }

// Value e of a tensor has word e mod 4 of the counter (e / 4, e / 2^34, 0, 0).
RG_HD inline Words value_words(uint64_t group, uint64_t seed) {
    return philox((uint32_t)group, (uint32_t)(group >> 32), 0u, 0u, seed);
}
// Attention's pair of query i and key j under head t (counted through the batch) has word j mod 4 of (j / 4, i, t, 1).
RG_HD inline Words pair_words(uint32_t key_group, uint32_t query, uint32_t head, uint64_t seed) {
    return philox(key_group, query, head, 1u, seed);
}

}  // namespace repro_dropout
