/*
 * repro_attention.h -- flat C ABI of the reproducible attention with its gradients and of the learned bias of
 * relative positions, on MI355X (gfx950).
 *
 * Queries q [B][Tq][H][D], keys and values k, v [B][Tk][KVH][D] (float32; any strides but the last, which is 1; query head h takes
 * key head h / (H / KVH)):
 *   t_ij = scale q_i . k_j + bias_h[j - i],   p_i = softmax of t_i over the keys that query i sees
 *   y_i = sum_j p_ij kept_ij / (1 - dropout) v_j
 * Query i of batch item b sees key j where j < key_lengths[b], with `causal` j <= i + query_start, and where the mask's bit is
 * set; one that sees none has y = 0 and takes no part in the gradients. What keys hold that no query sees, and what a
 * query and a key hold for each other where the one does not see the other, reaches nothing, NaN or not. A visible NaN or a score
 * past float32's range gives its row NaN; two scores of a row that are further apart than that range can give it, or its gradients, NaN. Scores are
 * counted in base 2, t_ij log2 e: one is past the range from 2.3e38 on, two can be apart by it from 1.1e38 on. A bias below
 * -6.9e29 (-infinity) counts as that.
 * The random bits of dropout are a function of the seed and the places of query and key (include/repro_dropout_math.h).
 *
 * Every operation is rounded once in a fixed order (include/repro_attention_math.h): the bits do not depend on the
 * device or the launch, and a row of y depends on its query and the keys it sees alone (and with dropout on their places), so that it
 * is the same computed alone, in a batch, or with padding.
 *
 * Plain C types only; the stream is a hipStream_t passed as void*. Return values are hipError_t
 * codes (0 success, 1 invalid value, others from the HIP runtime). Asynchronous, allocation-free.
 */
#ifndef REPRO_ATTENTION_H
#define REPRO_ATTENTION_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define RG_ATTENTION_MAX_D 128
#define RG_ATTENTION_MAX_LENGTH (1 << 22)
#define RG_ATTENTION_MAX_HEADS (1 << 20) /* B * H */
#define RG_ATTENTION_MAX_ROW (1 << 22)   /* H * D, and the strides of the positions */
#define RG_RELATIVE_BIAS_MAX_BORDERS 512

typedef struct rg_attention_config {
    long long B, Tq, Tk;
    int H, KVH, D; /* D 1 .. RG_ATTENTION_MAX_D, KVH a divisor of H */
    int causal;
    long long query_start; /* the keys' position that query 0 stands at */
    double scale, dropout; /* dropout in [0, 1) */
    unsigned long long seed;
    long long q_stride[3], k_stride[3], v_stride[3]; /* of the batch, the position and the head, in floats; not negative */
    long long mask_stride[3];                        /* of the batch, the head and the query, in words; 0: shared */
} rg_attention_config;

/* One item, one head, scale 1, no mask, no dropout; sizes 0. */
void rg_attention_config_init(rg_attention_config* cfg);

/* Truth values (bytes, not 0: seen) with the given numbers and strides (in bytes) of batch items, heads and queries, and Tk
 * keys key_stride apart, to words of 64 keys: word w of a row is at w, rows of (Tk + 63) / 64 words, contiguous
 * [items][heads][queries]. 1 (invalid value): null pointers, negative sizes, words off 8 bytes. */
int rg_attention_pack_mask(const unsigned char* mask, long long items, long long heads, long long queries, long long Tk,
                           const long long stride[3], long long key_stride, unsigned long long* words, void* stream);

/* The forward pass. key_lengths [B] (below 0 counts as 0, above Tk as Tk), mask (as packed above), relative_bias [H][Tq + Tk - 1] (the
 * distance j - i at column j - i + Tq - 1) and seed_at (the seed in device memory, read by the kernels, instead of
 * cfg->seed; used receives it) may be null. y [B][Tq][H][D] contiguous; stats [B][H][Tq][2] for the
 * backward pass, or null.
 * 1 (invalid value): null cfg, sizes out of range, scale not finite, dropout outside [0, 1); with rows and values to compute null q,
 * k, v or y, an address off 4 bytes (off 8: lengths, mask, stats, seeds), a workspace that is needed and null, off 16 bytes or too small; few
 * queries that make 2^32 or more blocks of 8 rows by 256 keys (which only keys of many items at one address, by a stride of 0, reach). */
int rg_attention_workspace(const rg_attention_config* cfg, int masked, size_t* bytes); /* masked: whether a mask is given */
int rg_attention_fp32(const rg_attention_config* cfg, const float* q, const float* k, const float* v,
                      const long long* key_lengths, const unsigned long long* mask, const float* relative_bias,
                      const unsigned long long* seed_at, unsigned long long* used, float* y, float* stats, void* workspace,
                      size_t workspace_bytes, void* stream);

/* The gradients for dy [B][Tq][H][D] (contiguous, as y): dq as y, dk and dv [B][Tk][KVH][D], drelative_bias as the bias;
 * dq, dk and dv are all written, drelative_bias where it is not null (the bias must be given then). seed_at is
 * what the forward pass left in `used`. Errors as above. */
int rg_attention_grad_workspace(const rg_attention_config* cfg, int want_bias, size_t* bytes);
int rg_attention_grad_fp32(const rg_attention_config* cfg, const float* dy, const float* q, const float* k, const float* v,
                           const long long* key_lengths, const unsigned long long* mask, const float* relative_bias,
                           const unsigned long long* seed_at, const float* y, const float* stats, float* dq, float* dk,
                           float* dv, float* drelative_bias, void* workspace, size_t workspace_bytes, void* stream);

/* The bias of relative positions by buckets: table [buckets][H], buckets = count + 1 (bidirectional: 2 (count + 1)), the bucket of a distance the
 * number of the ascending borders that it reaches (host memory). Key j is j - i - query_start away from query i; without
 * `both`, keys after the query count as at distance 0.
 * dense: out [H][Tq][Tk], else [H][Tq + Tk - 1] (as rg_attention_fp32 takes it). The gradient's dout likewise; its
 * workspace is only needed for a dense one.
 * 1 (invalid value): sizes out of range, borders null, not ascending or not positive, null pointers, a workspace too small. */
typedef struct rg_relative_bias_config {
    long long Tq, Tk, query_start;
    int H, count, both, dense;
    const int* borders;
} rg_relative_bias_config;

int rg_relative_bias_fp32(const rg_relative_bias_config* cfg, const float* table, float* out, void* stream);
int rg_relative_bias_grad_workspace(const rg_relative_bias_config* cfg, size_t* bytes);
int rg_relative_bias_grad_fp32(const rg_relative_bias_config* cfg, const float* dout, float* dtable, void* workspace,
                               size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
