#pragma once
// What defines the reproducible norms: every value's operations, one IEEE float32 rounding each in a
// fixed order (build without -ffast-math and without FP contraction), and the order of every sum.
//
// Sum over a row of D values: chunks of 4 consecutive values (missing ones +0) give
// (v0 + v1) + (v2 + v3); chunk c goes to strand c mod S, S = 256 for D <= 4096, else 1024, in ascending
// order from the strand's first chunk (a strand without chunks is +0). Strands s, s + 64, s + 128, ...
// are added as a balanced tree of neighbours, which leaves 64 values, and these as a balanced tree
// whose first level adds l and l + 32, the next l and l + 16, and so on.
//
// Sum over rows (the gradients of weights, biases and gates): see Partition.

#include "repro_gemm_math.h"

namespace repro_norm {

constexpr int MAX_D = 16384;

RG_HD inline int strands_of(int D) { return D <= 4096 ? 256 : 1024; }

// Rows are divided into sections, a section's rows into strands of at most `rows` consecutive ones, each
// added up in ascending order from +0. `join` neighbouring strands of a section (missing ones +0) are added as a
// balanced tree to a partial; a sum over partials adds those with equal p mod 16 in ascending order
// from +0, and the 16 results as a balanced tree of neighbours.
// A gate of G rows has a gradient row for each group of N / G rows. Where groups are at least as long as a
// strand, a section is a group, and its gate's gradient is the sum of its partials. Else there is one
// section, a strand holds whole groups, and adds up each group's gradient by itself.
// Strands are short enough to give a GPU work and long enough that their partials are little to
// write beside the rows; they depend on the sizes alone, so the results do too. There are at most 2 * aim partials
// (below) and `aim` sections: groups are sections only where they are at least as long as N / aim.
struct Partition {
    long long sections, section_rows;  // the last section may be shorter only where it is the only one
    int rows, join;
    long long strands, partials;  // per section
    bool gate_inside;             // groups within strands
    long long group_rows;
};

inline Partition partition(long long N, int D, long long G) {
    Partition p;
    p.join = D <= 1024 ? 4 : 1;
    const long long aim = D <= 1024 ? 2048 : 512;
    const long long rows = (N + aim - 1) / aim;
    p.rows = (int)(rows > 4 ? rows : 4);
    p.group_rows = G > 0 ? N / G : N;
    p.gate_inside = G > 1 && p.group_rows < p.rows;
    if (p.gate_inside) p.rows = (int)(p.rows / p.group_rows * p.group_rows);
    p.sections = p.gate_inside || G < 1 ? 1 : G;
    p.section_rows = p.sections > 1 ? p.group_rows : N;
    p.strands = (p.section_rows + p.rows - 1) / p.rows;
    p.partials = (p.strands + p.join - 1) / p.join;
    return p;
}

// ---- the values' operations ----

struct RowStats {
    float mean, rstd;  // mean 0 for an RMS norm
};

RG_HD inline float centred(float v, float mean, bool layer) { return layer ? v - mean : v; }
RG_HD inline float mean_of(float sum, int D) { return sum / (float)D; }
RG_HD inline float rstd_of(float square_sum, int D, float eps) {
    return 1.0f / __builtin_sqrtf(square_sum / (float)D + eps);
}
// hat: the normalised value; null weights are left out
RG_HD inline float affine(float hat, bool weighted, float w, bool biased, float b) {
    const float y = weighted ? hat * w : hat;
    return biased ? y + b : y;
}
// d: the gradient of the normalised value, c1 and c2 the row's means of d and of d * hat
RG_HD inline float backward(float d, float hat, float rstd, float c1, float c2, bool layer) {
    const float e = layer ? d - c1 : d;
    return (e - hat * c2) * rstd;
}

}  // namespace repro_norm
