/*
 * repro_loss.h -- flat C ABI of the reproducible softmax cross entropy of a vocabulary projection
 * (a language model's head) with its gradients, on MI355X (gfx950).
 *
 * For hidden states x [N][D], a weight w [V][D] (float32, row-major, contiguous) and target words
 * t [N] (int64):
 *   z = x w^T,   loss_n = ln(sum_v e^(z_nv)) - z_n,t_n
 *   dz_nv = g_n (softmax(z_n)_v - [v = t_n]),   dx = dz w,   dw = dz^T x
 * A target equal to ignore_index leaves its token out (loss and gradients 0); another one outside
 * [0, V) gives the token a loss of NaN and no gradients. The losses are reduced to their sum, their
 * mean over the tokens that count (0 of them: NaN), or not; g_n is 1, 1 / count, or the caller's.
 * A token whose row of x holds a NaN or an infinity, or whose largest logit is one, has a NaN loss, a NaN row of dx, and
 * makes its target's row of dw NaN; where w holds one, that is so for every token. Nothing that the rows of tokens
 * that do not count hold reaches loss, dw or the other tokens' dx.
 *
 * The three products are the reproducible GEMM's (S int8 slices); the target word's share of the
 * gradients, g_n (softmax - 1), stays out of dz there, where it would set the scale that the other words'
 * small shares are rounded at, and is added in float32. Every other operation is rounded once in a
 * fixed order (include/repro_loss_math.h), so the bits do not depend on the device or the launch.
 * The logits are never kept: tokens are taken in groups (RG_LOSS_* below), each of which goes from
 * its logits to its share of the gradients, in one product for each of z, dx and dw.
 *
 * Plain C types only; the stream is a hipStream_t passed as void*. Return values are hipError_t
 * codes (0 success, 1 invalid value, 801 not supported, others from the HIP runtime). Asynchronous,
 * allocation-free.
 */
#ifndef REPRO_LOSS_H
#define REPRO_LOSS_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { RG_LOSS_MEAN = 0, RG_LOSS_SUM = 1, RG_LOSS_NONE = 2 };

#define RG_LOSS_MAX_TOKENS (1 << 22)
#define RG_LOSS_MAX_SIZE (1 << 23)
#define RG_LOSS_MAX_WORDS (1 << 25) /* 64 threads a word are the most of a launch, fewer than 2^32 */

typedef struct rg_loss_config {
    long long N;            /* tokens, 0 .. RG_LOSS_MAX_TOKENS */
    int D, V;               /* 1 .. RG_LOSS_MAX_SIZE and 1 .. RG_LOSS_MAX_WORDS, and what the GEMM takes
                             * as its inner length: at S = 3 about 1,000,000 */
    int slices;             /* S in 1..3 */
    int reduction;          /* RG_LOSS_* */
    long long ignore_index;
} rg_loss_config;

/* Three slices, the mean, ignore_index -100; sizes 0. */
void rg_loss_config_init(rg_loss_config* cfg);

/* Tokens of a group for a vocabulary of V words: a power of two from 128 to 2048, of at most 2^27 logits
 * where it is past 128. 0 for V < 1. */
int rg_loss_group_tokens(int V);

/* Bytes that rg_linear_cross_entropy needs for these sizes; want_dx, want_dw: whether it is asked for
 * the gradient. Queries the current device. Errors as below. */
int rg_linear_cross_entropy_workspace(const rg_loss_config* cfg, int want_dx, int want_dw, size_t* bytes);

/* loss: one float, or N for RG_LOSS_NONE; dx [N][D]; dw [V][D]; each may be null. factors (N floats, may
 * be null): g_n instead of the reduction's. N = 0: loss 0 (the mean NaN), dw zero.
 * 1 (invalid value): null cfg, sizes, slices or reduction out of range; with N > 0 null x, w or target, an
 * address off 4 bytes (off 8: target), or a workspace that is null, off 256 bytes or too small. */
int rg_linear_cross_entropy(const rg_loss_config* cfg, const float* x, const float* w, const long long* target,
                            const float* factors, float* loss, float* dx, float* dw, void* workspace,
                            size_t workspace_bytes, void* stream);

/* The nx floats of x and the ny of y times factor[0], in device memory; nothing is written where it is 1 (the
 * gradients of a loss that is not scaled further). 1 (invalid value): null pointers to what is to be scaled. */
int rg_scale_fp32(float* x, size_t nx, float* y, size_t ny, const float* factor, void* stream);

#ifdef __cplusplus
}
#endif
#endif
