/* Launchers of the batched serving operators (include/lunelette_serving.h):
 * called with checked arguments, 0 or the HIP error of a refused launch. */
#ifndef LH_SERVING_H
#define LH_SERVING_H

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#include "lunelette_serving.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A multiple of 16 that holds `bytes`. */
static inline size_t lh_round16(size_t bytes)
{
    return (bytes + 15) & ~(size_t)15;
}

int lh_launch_q4_pack(const uint8_t *codes, const uint16_t *scales, uint32_t rows, uint32_t cols,
    uint32_t group, uint8_t *packed, hipStream_t s);
int lh_launch_q4_quantize(const float *w, uint32_t rows, uint32_t cols, uint32_t group,
    uint8_t *packed, hipStream_t s);
int lh_launch_q4_matvec(const uint8_t *packed, const float *x, size_t x_stride, float *y,
    size_t y_stride, uint32_t rows, uint32_t cols, uint32_t group, uint32_t tokens,
    uint8_t *scratch, hipStream_t s);

int lh_launch_logprobs(const float *logits, size_t stride, uint32_t rows, uint32_t vocab,
    const int64_t *tokens, float *logprob, float *entropy, uint32_t top, int64_t *top_ids,
    float *top_logprobs, uint8_t *scratch, hipStream_t s);

typedef struct {
    const float *q, *k, *v, *cosine, *sine, *qfactor;
    float *q_out;
    size_t q_stride, k_stride, v_stride, q_out_stride;
    uint32_t group, positions; /* query heads of a KV head; rows of the rotation */
} lh_append_rows;
int lh_launch_paged_append(const lh_paged_cache *cache, const lh_paged_batch *batch,
    const lh_append_rows *rows, hipStream_t s);
int lh_launch_paged_read(const lh_paged_cache *cache, const lh_paged_batch *batch, float *keys,
    size_t k_stride, float *values, size_t v_stride, hipStream_t s);
int lh_launch_paged_attention(const lh_paged_cache *cache, const lh_paged_batch *batch,
    uint32_t group, const float *q, size_t q_stride, float scale, float *out, size_t out_stride,
    uint8_t *scratch, hipStream_t s);

/* Scratch of the launchers above, from the sizes alone. */
size_t lh_q4_scratch_bytes(uint32_t cols, uint32_t tokens);
size_t lh_logprobs_scratch_bytes(uint32_t rows, uint32_t vocab, uint32_t top);
size_t lh_paged_attention_scratch_bytes(const lh_paged_cache *cache, const lh_paged_batch *batch,
    uint32_t group);

#ifdef __cplusplus
}
#endif

#endif
