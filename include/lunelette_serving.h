/* Operators of batched serving from little memory (no counterpart in the
 * reference): a paged KV cache of several sequences in FP16 rows or 4-bit
 * codes with the append and the attention that use it, products with 4-bit
 * weights, and log probabilities of logit rows.
 *
 * The conventions are those of lunelette_kernels.h: pointers named d_* are
 * device pointers on the current device, `stream` is a hipStream_t passed as
 * void* (NULL = the null stream), calls return 0 or -1 (lh_last_error()
 * describes the refusal, and nothing was launched). Activations and logits are
 * FP32. No call allocates, synchronizes or keeps state between calls, so all
 * may be captured into a graph. A call's scratch holds nothing before or after
 * it; calls that may run at the same time (other streams, two graphs) need
 * scratch of their own. FP32 tensors need 4-byte alignment only (rows on
 * 16-byte boundaries load faster); scratch, packed weights and pages need 16.
 */
#ifndef LUNELETTE_SERVING_H
#define LUNELETTE_SERVING_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- 4-bit weights with group scales ----
 * w[r][c] = scale[r][c / group] * (code[r][c] - 8), code 0..15, scale BF16;
 * group 32, 64 or 128, cols a multiple of it up to 65536, rows 1..2^20. */

/* Bytes of packed weights (16-row tiles in the order in which the matrix
 * instructions take them); 0 for sizes outside the ranges above. */
size_t lh_q4_bytes(size_t rows, size_t cols, size_t group);
/* Lays out d_codes [rows][cols / 2] (two codes to a byte, the even column in
 * the low bits) and d_scales [rows][cols / group] as packed weights. */
int lh_q4_pack(const uint8_t *d_codes, const uint16_t *d_scales, size_t rows, size_t cols,
    size_t group, void *d_packed, void *stream);
/* Packs d_w [rows][cols] FP32 by rounding: scale = bf16(max |w| / 7 over the
 * group), code = 8 + rint(w / scale) within 1..15. A group whose scale rounds to
 * zero has code 8 everywhere; one with a nonfinite weight a NaN scale. */
int lh_q4_quantize(const float *d_w, size_t rows, size_t cols, size_t group, void *d_packed,
    void *stream);
/* Scratch bytes of lh_q4_matvec at these sizes for any number of rows (0: none is
 * needed). */
size_t lh_q4_scratch(size_t cols, size_t tokens);
/* y[t][r] = sum_c w[r][c] x[t][c] for 1..65535 tokens; rows of x and y are
 * x_stride and y_stride elements apart (x_stride >= cols, y_stride >= rows).
 * Products are formed from x as two FP16 planes scaled by a power of two per
 * token, or per token and 128 columns (each x to 2^-22 of itself or 2^-38 of
 * its row's largest), sums are FP32, which scales below 2^102 stay in. A row of x
 * with an Inf or NaN gives NaN in its row of y. y must not overlap x. */
int lh_q4_matvec(const void *d_packed, const float *d_x, size_t x_stride, float *d_y,
    size_t y_stride, size_t rows, size_t cols, size_t group, size_t tokens, void *d_scratch,
    size_t scratch_bytes, void *stream);

/* ---- log probabilities ---- */

#define LH_LOGPROBS_TOP 64

/* Scratch bytes of lh_logprobs; 0 for sizes that it refuses. */
size_t lh_logprobs_scratch(size_t rows, size_t vocab, size_t top);
/* For each of rows (1..65535) logit rows of vocab (1..2^24) values, stride >=
 * vocab elements apart, with p = softmax(row):
 * - d_logprob [rows]: ln p of the row's token in d_tokens [rows]; 0 for token
 *   -1 (no token), NaN for any other id outside [0, vocab). Both NULL: none.
 * - d_entropy [rows]: -sum p ln p in nats. NULL: none.
 * - d_top_ids, d_top_logprobs [rows][top], top 0..LH_LOGPROBS_TOP: the likeliest
 *   ids and their ln p in falling order, equal logits by lower id (-0 equals
 *   +0). Places past the row's unmasked tokens hold id -1 and
 *   -Inf.
 * A logit of -Inf is a masked token: p = 0, ln p = -Inf, no part in the
 * entropy. A row of nothing else has no distribution: ln p -Inf, entropy 0, no
 * top tokens. A row with a NaN or +Inf gives NaN everywhere and ids of -1.
 * The sums are formed in 64 bits. */
int lh_logprobs(const float *d_logits, size_t stride, size_t rows, size_t vocab,
    const int64_t *d_tokens, float *d_logprob, float *d_entropy, size_t top, int64_t *d_top_ids,
    float *d_top_logprobs, void *d_scratch, size_t scratch_bytes, void *stream);

/* ---- paged KV cache ---- */

enum {
    LH_CACHE_F16 = 0, /* rows rounded to FP16 (from 65520 on Inf) */
    /* per (position, KV head) vector of keys or values 4-bit codes and a BF16
     * scale and zero: zero = bf16(min), scale = bf16((max - zero) / 15),
     * code = rint((v - zero) / scale) within 0..15, value = scale * code + zero.
     * A vector with an Inf or NaN, or one whose scale or zero overflows, reads
     * as NaN throughout. */
    LH_CACHE_Q4 = 1
};

/* One layer's cache: `pages` pages of page_size positions (a multiple of 32 up
 * to 1024), kv_heads 1..64, head_dim 64 or 128. d_pages holds
 * lh_paged_cache_bytes() bytes; the order inside a page is the library's own.
 * Pages need no clearing before their first use. */
typedef struct {
    int kind;
    uint32_t kv_heads, head_dim, page_size, pages;
    void *d_pages;
} lh_paged_cache;
size_t lh_paged_cache_bytes(const lh_paged_cache *cache);

/* The sequences of a call. Sequence s owns the token rows d_query_start[s] ..
 * d_query_start[s + 1] - 1 of the call's tensors (d_query_start
 * [sequences + 1], not falling, within 0..tokens; rows behind the last one stay
 * as they are), which are its last positions: d_length[s] counts its positions
 * with them. Position p lies in page d_table[s][p / page_size] (rows of
 * table_width ids). The three arrays are read on the device, so a captured
 * call follows them; max_query and max_length size the launch and should bound
 * a sequence's rows and length (larger ones are computed too, only slower).
 * sequences 1..65535, tokens 1..2^24, table_width 1..2^20.
 * A token whose position is negative, past the table or in a page id outside
 * [0, pages) has no place in the cache: it is not appended and reads as NaN. */
typedef struct {
    uint32_t sequences, tokens, table_width, max_query, max_length;
    const int32_t *d_query_start, *d_length, *d_table;
} lh_paged_batch;

/* Appends the call's keys and values (rows of d_k, d_v [tokens][kv_heads *
 * head_dim], k_stride and v_stride elements apart), keys rotated on the way by
 * the rows of their positions in d_cos, d_sin [positions][head_dim] (as
 * lh_yarn writes them: split halves, both halves of a row alike), and writes
 * the rotated queries, times d_qfactor[position] where that is not NULL, to
 * d_q_out (which may be d_q with the same stride, and otherwise shares no element
 * with another tensor).
 * heads is a multiple of kv_heads up to 64 of them each; 0 leaves the queries
 * and d_qfactor out. d_cos and d_sin NULL: rotated already. The rotation is formed
 * in 64 bits and rounded to FP32 (for 4-bit codes not at all) before the cache's
 * format.
 * With d_cos or d_qfactor a token whose position is negative or not below
 * `positions` is not appended and its query row is NaN; without them that holds
 * for negative positions. A page that a call appends to must stand in one place
 * of one sequence's table. */
int lh_paged_append(const lh_paged_cache *cache, const lh_paged_batch *batch, uint32_t heads,
    const float *d_q, size_t q_stride, const float *d_k, size_t k_stride, const float *d_v,
    size_t v_stride, const float *d_cos, const float *d_sin, uint32_t positions,
    const float *d_qfactor, float *d_q_out, size_t q_out_stride, void *stream);
/* Reads the cache rows of the call's tokens back as FP32 rows (the paged
 * counterpart of lunelette_metal_read_kv); d_keys or d_values may be NULL. */
int lh_paged_read(const lh_paged_cache *cache, const lh_paged_batch *batch, float *d_keys,
    size_t k_stride, float *d_values, size_t v_stride, void *stream);
/* Scratch bytes of lh_paged_attention (0: none is needed or bad arguments). */
size_t lh_paged_attention_scratch(const lh_paged_cache *cache, const lh_paged_batch *batch,
    uint32_t heads);
/* Causal attention of the call's tokens, appended before: query head h of
 * d_q [tokens][heads * head_dim] over the positions up to its token's own of
 * KV head h / (heads / kv_heads), scores times scale (positive and finite),
 * into d_out (which must not overlap d_q). A token at a negative position sees
 * nothing and gives 0; one that sees a position without a place in the cache
 * gives NaN, as does one that sees a key with an Inf or NaN, or a value with one
 * (in FP16 pages in that element alone). What no token sees may hold anything.
 * Products are formed from two FP16 planes: of queries, which keep them to 2^-22
 * of themselves or 2^-38 of their row's largest, and of probabilities (in 4-bit
 * pages times their values' scales), 2^-22 of themselves or 2^-32 of the row's
 * largest of these. Sums and the softmax are FP32: scores, and a row's number of
 * positions times its largest value, have to lie in its range. 4-bit keys count to
 * 2^-125. */
int lh_paged_attention(const lh_paged_cache *cache, const lh_paged_batch *batch, uint32_t heads,
    const float *d_q, size_t q_stride, float scale, float *d_out, size_t out_stride,
    void *d_scratch, size_t scratch_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif
