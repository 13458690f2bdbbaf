/*
 * repro_adamw.h -- flat C ABI of the reproducible AdamW step over many tensors on MI355X (gfx950).
 *
 * For every value p of every tensor, with its gradient g and moments m, v (all float32):
 *   m <- m beta1 + g (1 - beta1)           v <- v beta2 + g g (1 - beta2)
 *   p <- p (1 - lr weight_decay) - m / (sqrt(v) / sqrt(1 - beta2^step) + eps) * lr / (1 - beta1^step)
 * each operation rounded once in the order of include/repro_adamw_math.h, so the bits do not depend
 * on the device, the launch or how the tensors are listed. Non-finite gradients give what these
 * operations give.
 *
 * Plain C types only; the stream is a hipStream_t passed as void*. Return values are hipError_t
 * codes (0 success, 1 invalid value, others from the HIP runtime). Asynchronous, allocation-free;
 * the tensor list is read before the call returns. A step's constants are launch arguments: a
 * captured graph repeats the captured step.
 */
#ifndef REPRO_ADAMW_H
#define REPRO_ADAMW_H

#ifdef __cplusplus
extern "C" {
#endif

typedef struct rg_adamw_config {
    double lr, beta1, beta2, eps, weight_decay;
    long long step; /* the step being taken: 1 for the first */
} rg_adamw_config;

/* lr 1e-3, betas 0.9 and 0.999, eps 1e-8, weight decay 1e-2, step 1. */
void rg_adamw_config_init(rg_adamw_config* cfg);

/* One tensor: n values each of p, g, m and v, contiguous, overlapping nothing else in the list. */
typedef struct rg_adamw_tensor {
    float* p;
    const float* g;
    float* m;
    float* v;
    long long n; /* 0: nothing is done for this tensor */
} rg_adamw_tensor;

/* 1 (invalid value): null cfg, a null list or count < 0, n < 0, a null pointer with n > 0, a
 * pointer off 4 bytes; betas outside [0, 1), lr, eps or weight_decay negative or NaN, step < 1. */
int rg_adamw_fp32(const rg_adamw_tensor* tensors, int count, const rg_adamw_config* cfg, void* stream);

/* The moments in 8 bits: blocks of RG_ADAMW8_BLOCK consecutive values share an exponent
 * (include/repro_adamw_math.h). For a tensor of n values, with b = ceil(n / RG_ADAMW8_BLOCK), m and
 * v hold b * RG_ADAMW8_BLOCK codes and m_exp and v_exp b exponents; all zero is the state before
 * the first step. The codes past n are written as zero. m and v at addresses that are multiples of 4. */
#define RG_ADAMW8_BLOCK 256
typedef struct rg_adamw8_tensor {
    float* p;
    const float* g;
    unsigned char* m;
    unsigned char* m_exp;
    unsigned char* v;
    unsigned char* v_exp;
    long long n;
} rg_adamw8_tensor;

/* Errors as rg_adamw_fp32. The moments' rounding numbers go by the step and a value's position,
 * counted over the list with each tensor starting at a whole block. */
int rg_adamw8_fp32(const rg_adamw8_tensor* tensors, int count, const rg_adamw_config* cfg, void* stream);

/* The values that `blocks` blocks of codes stand for: m_values and v_values of blocks *
 * RG_ADAMW8_BLOCK floats. 1 (invalid value): a null pointer with blocks > 0, codes off 4 bytes,
 * values off 16 bytes, blocks < 0 or past 2^31 - 1. */
int rg_adamw8_values(const unsigned char* m, const unsigned char* m_exp, const unsigned char* v,
                     const unsigned char* v_exp, float* m_values, float* v_values, long long blocks,
                     void* stream);

#ifdef __cplusplus
}
#endif
#endif
