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

/* What the rows that are rounded to 8 bits are made of: x; SiLU(x) * second; or
 * gamma times the normalized x + second (NULL: x), the sum kept in `sum` or not. */
enum { LH_Q8_ROWS, LH_Q8_SILU, LH_Q8_NORM };
typedef struct {
    const float *x, *second, *gamma;
    float *sum, *scales;
    int8_t *codes;
    size_t x_stride, second_stride, sum_stride, code_stride;
    uint32_t width, tokens;
} lh_q8_source;
int lh_launch_q8_rows(int kind, const lh_q8_source *rows, hipStream_t s);
int lh_launch_q8_pack(const int8_t *codes, const float *scales, uint32_t rows, uint32_t cols,
    uint8_t *packed, hipStream_t s);
int lh_launch_q8_quantize(const float *w, uint32_t rows, uint32_t cols, uint8_t *packed,
    hipStream_t s);
int lh_launch_q8_matvec(const uint8_t *packed, const int8_t *x, size_t x_stride,
    const float *x_scales, float *y, size_t y_stride, uint32_t rows, uint32_t cols,
    uint32_t tokens, uint8_t *scratch, hipStream_t s);
/* The kernel that lh_launch_q8_matvec takes at these sizes, and its column splits. */
int lh_q8_way(uint32_t rows, uint32_t cols, uint32_t tokens, uint32_t *splits);

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

typedef struct {
    const float *logits, *scores;
    const uint8_t *done;
    int32_t *parent;
    int64_t *token, stop;
    float *score;
    uint8_t *done_out;
    size_t stride;
    uint32_t groups, beams, vocab, keep;
} lh_beam_choice;
int lh_launch_beam_select(const lh_beam_choice *choice, uint8_t *scratch, hipStream_t s);
enum { LH_BEAM_LAYERS = 64 }; /* caches of a reordering */
int lh_launch_beam_reorder(const lh_paged_cache *caches, uint32_t layers, uint32_t groups,
    uint32_t beams, const int32_t *parent, const int32_t *length, const int32_t *table,
    int32_t *table_out, uint32_t width, hipStream_t s);

/* Scratch of the launchers above, from the sizes alone. */
size_t lh_q4_scratch_bytes(uint32_t cols, uint32_t tokens);
size_t lh_q8_scratch_bytes(uint32_t rows, uint32_t cols, uint32_t tokens);
size_t lh_beam_scratch_bytes(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t keep);
size_t lh_logprobs_scratch_bytes(uint32_t rows, uint32_t vocab, uint32_t top);
size_t lh_paged_attention_scratch_bytes(const lh_paged_cache *cache, const lh_paged_batch *batch,
    uint32_t group);

#ifdef __cplusplus
}
#endif

#endif
