/*
 * repro_dropout.h -- flat C ABI of the reproducible dropout on MI355X (gfx950).
 *
 * y = x / (1 - p) where a value is kept, 0 (whatever x holds there) where it is dropped, each with probability p by random
 * bits that are a function of a seed and the value's place (include/repro_dropout_math.h): the same on every
 * run, device and launch. The same call with the gradient of y for x is its gradient; no mask is stored.
 *
 * Plain C types only; the stream is a hipStream_t passed as void*. Return values are hipError_t
 * codes (0 success, 1 invalid value, others from the HIP runtime). Asynchronous, allocation-free.
 */
#ifndef REPRO_DROPOUT_H
#define REPRO_DROPOUT_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* n floats; y may be x. seed_at, when not null, is the seed in device memory, read when the kernel runs (so a captured
 * graph may be given another one for each replay), instead of `seed`; used, when not null, receives the seed that was read.
 * 1 (invalid value): p outside [0, 1) or NaN; with n > 0 null x or y, one off 4 bytes, seed_at or used off 8. */
int rg_dropout_fp32(const float* x, float* y, size_t n, double p, unsigned long long seed,
                    const unsigned long long* seed_at, unsigned long long* used, void* stream);

#ifdef __cplusplus
}
#endif
#endif
