/*
 * repro_norm.h -- flat C ABI of the reproducible residual addition with the norms before and after a
 * block, on MI355X (gfx950).
 *
 * For N rows of D float32 values, row-major and contiguous:
 *   r = x + scale * (gate * u),  u = Norm(f) * post_weight + post_bias  (post), else f
 *   y = Norm(r) * weight + bias
 * Norm is a layer norm, (v - mean) / sqrt(mean((v - mean)^2) + eps), or an RMS norm,
 * v / sqrt(mean(v^2) + eps). Absent: a null gate, weight or bias; a null f stands for the norm of x alone
 * (r = x is not written). The gate has gate_rows rows of D values, gate_rows a divisor of N: row n of x
 * takes row n / (N / gate_rows) of it (1: one for each channel; N: one for each value).
 *
 * Every operation is rounded once in a fixed order, and every sum's order is fixed by the sizes
 * (include/repro_norm_math.h): the bits do not depend on the device or the launch. A row holding a NaN or
 * infinity affects its own r, y and gradients (and the sums over rows) only.
 *
 * Plain C types only; the stream is a hipStream_t passed as void*. Return values are hipError_t
 * codes (0 success, 1 invalid value, others from the HIP runtime). Asynchronous, allocation-free.
 */
#ifndef REPRO_NORM_H
#define REPRO_NORM_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define RG_NORM_MAX_D 16384

typedef struct rg_norm_config {
    long long N;
    int D;               /* 1 .. RG_NORM_MAX_D */
    int rms;             /* 0: layer norms, 1: RMS norms */
    int post;            /* f is normalised first */
    long long gate_rows; /* 0: no gate */
    float eps, scale;
} rg_norm_config;

/* A layer norm with eps 1e-5, scale 1, no post norm, no gate; N and D 0. */
void rg_norm_config_init(rg_norm_config* cfg);

/* The forward pass. stats: N * 4 floats (mean and 1 / deviation of r, then of f) for the backward pass,
 * or null. r null exactly where f is. flag, when not null, is lowered to op_id if a norm of a row of r (post: or of f)
 * is not finite (a NaN or infinity in the row, or squares past float32's range).
 * 1 (invalid value): null cfg, x or y; N < 0, D out of range, eps negative or NaN; f and r not null together; a post
 * norm or gate without f, gate_rows not a divisor of N, or gate and gate_rows not given together. */
int rg_residual_norm_fp32(const rg_norm_config* cfg, const float* x, const float* f, const float* gate,
                          const float* post_weight, const float* post_bias, const float* weight,
                          const float* bias, float* r, float* y, float* stats, int* flag, int op_id,
                          void* stream);

/* The gradients. dr and dy: of r and y, one of them may be null (all zero); r (x where f is null), f and
 * stats as in the forward pass. Each output may be null: dx, df [N][D], dgate [gate_rows][D], and the
 * weights' and biases' [D]. The workspace holds at least the given bytes (0 where no sum over rows is
 * asked for: sums = 0). flag as above, where a value of dx is not finite.
 * 1 (invalid value): as above; dr and dy both null, an output whose input is absent, stats off 16 bytes (in
 * either pass), a workspace that is needed and null, too small or off 4 bytes. */
int rg_residual_norm_grad_workspace(const rg_norm_config* cfg, int sums, size_t* bytes);
int rg_residual_norm_grad_fp32(const rg_norm_config* cfg, const float* dr, const float* dy, const float* r,
                               const float* f, const float* gate, const float* post_weight,
                               const float* post_bias, const float* weight, const float* stats, float* dx,
                               float* df, float* dgate, float* dpost_weight, float* dpost_bias,
                               float* dweight, float* dbias, void* workspace, size_t workspace_bytes,
                               int* flag, int op_id, void* stream);

#ifdef __cplusplus
}
#endif
#endif
