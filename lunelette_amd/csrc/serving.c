/* Batched serving operators (include/lunelette_serving.h): argument checks and
 * launches. Whatever the host can see is refused here, before any launch; the
 * arrays of a batch are read on the device, whose kernels bound them. */
#include "lunelette_serving.h"
#include "lh_internal.h"
#include "lh_serving.h"

#include <math.h>

static int launched(int status, const char *what)
{
    if (status) {
        lh_set_error("%s launch failed: %s", what, lh_launch_text(status));
        return -1;
    }
    return 0;
}

static int refuse(const char *what)
{
    lh_set_error("%s", what);
    return -1;
}

static int aligned(const void *ptr, uintptr_t bytes)
{
    return ((uintptr_t)ptr & (bytes - 1)) == 0;
}

/* Row strides stay below 2^36 elements (256 GiB), so no offset of 2^24 rows passes
 * 64 bits. */
static int stride_ok(size_t stride, size_t width)
{
    return stride >= width && stride <= ((size_t)1 << 36);
}

/* ---- 4-bit weights ---- */

static int q4_sizes(size_t rows, size_t cols, size_t group)
{
    return rows && rows <= ((size_t)1 << 20) && cols && cols <= 65536 &&
        (group == 32 || group == 64 || group == 128) && cols % group == 0;
}

size_t lh_q4_bytes(size_t rows, size_t cols, size_t group)
{
    if (!q4_sizes(rows, cols, group)) {
        return 0;
    }
    return (rows + 15) / 16 * ((cols + 127) / 128) * (1024 + 32 * (128 / group));
}

int lh_q4_pack(const uint8_t *d_codes, const uint16_t *d_scales, size_t rows, size_t cols,
    size_t group, void *d_packed, void *stream)
{
    if (!d_codes || !d_scales || !d_packed || !q4_sizes(rows, cols, group) ||
        !aligned(d_packed, 16) || !aligned(d_scales, 2)) {
        return refuse("q4_pack: require pointers (packed on 16 bytes), rows 1..2^20, group 32, 64 "
            "or 128, cols a multiple of it up to 65536");
    }
    return launched(lh_launch_q4_pack(d_codes, d_scales, (uint32_t)rows, (uint32_t)cols,
        (uint32_t)group, d_packed, (hipStream_t)stream), "q4 pack");
}

int lh_q4_quantize(const float *d_w, size_t rows, size_t cols, size_t group, void *d_packed,
    void *stream)
{
    if (!d_w || !d_packed || !q4_sizes(rows, cols, group) || !aligned(d_packed, 16) ||
        !aligned(d_w, 4)) {
        return refuse("q4_quantize: require pointers (packed on 16 bytes), rows 1..2^20, group "
            "32, 64 or 128, cols a multiple of it up to 65536");
    }
    return launched(lh_launch_q4_quantize(d_w, (uint32_t)rows, (uint32_t)cols, (uint32_t)group,
        d_packed, (hipStream_t)stream), "q4 quantize");
}

size_t lh_q4_scratch(size_t cols, size_t tokens)
{
    if (!cols || cols > 65536 || !tokens || tokens > 65535) {
        return 0;
    }
    return lh_q4_scratch_bytes((uint32_t)cols, (uint32_t)tokens);
}

int lh_q4_matvec(const void *d_packed, const float *d_x, size_t x_stride, float *d_y,
    size_t y_stride, size_t rows, size_t cols, size_t group, size_t tokens, void *d_scratch,
    size_t scratch_bytes, void *stream)
{
    if (!d_packed || !d_x || !d_y || !q4_sizes(rows, cols, group) || !tokens || tokens > 65535 ||
        !aligned(d_packed, 16) || !aligned(d_x, 4) || !aligned(d_y, 4)) {
        return refuse("q4_matvec: require pointers (packed on 16 bytes), rows 1..2^20, group 32, "
            "64 or 128, cols a multiple of it up to 65536, tokens 1..65535");
    }
    if (!stride_ok(x_stride, cols) || !stride_ok(y_stride, rows)) {
        return refuse("q4_matvec: x_stride below cols or y_stride below rows");
    }
    const size_t need = lh_q4_scratch_bytes((uint32_t)cols, (uint32_t)tokens);
    if (need && (!d_scratch || scratch_bytes < need || !aligned(d_scratch, 16))) {
        lh_set_error("q4_matvec: needs %zu bytes of scratch on a 16-byte boundary", need);
        return -1;
    }
    if ((const void *)d_x == (const void *)d_y) {
        return refuse("q4_matvec: y must not overlap x");
    }
    return launched(lh_launch_q4_matvec(d_packed, d_x, x_stride, d_y, y_stride, (uint32_t)rows,
        (uint32_t)cols, (uint32_t)group, (uint32_t)tokens, d_scratch, (hipStream_t)stream),
        "q4 matvec");
}

/* ---- 8-bit rows and weights ---- */

static int q8_codes_ok(const int8_t *d_codes, size_t code_stride, const float *d_scales,
    size_t width, size_t tokens)
{
    return d_codes && d_scales && width && width <= 65536 && tokens && tokens <= 65535 &&
        aligned(d_codes, 16) && aligned(d_scales, 4) && code_stride % 16 == 0 &&
        stride_ok(code_stride, width);
}

static int q8_codes_refused(const int8_t *d_codes, size_t code_stride, const float *d_scales,
    size_t width, size_t tokens, const char *what)
{
    if (!q8_codes_ok(d_codes, code_stride, d_scales, width, tokens)) {
        lh_set_error("%s: require codes in rows on 16-byte boundaries with their scales, width "
            "1..65536, tokens 1..65535", what);
        return 1;
    }
    return 0;
}

int lh_q8_rows(const float *d_x, size_t x_stride, size_t width, size_t tokens, int8_t *d_codes,
    size_t code_stride, float *d_scales, void *stream)
{
    if (q8_codes_refused(d_codes, code_stride, d_scales, width, tokens, "q8_rows")) {
        return -1;
    }
    if (!d_x || !aligned(d_x, 4) || !stride_ok(x_stride, width)) {
        return refuse("q8_rows: x in rows of the width required");
    }
    if ((const void *)d_x == (const void *)d_codes || d_x == d_scales) {
        return refuse("q8_rows: codes and scales must not overlap x");
    }
    const lh_q8_source rows = {
        .x = d_x, .x_stride = x_stride, .scales = d_scales, .codes = d_codes,
        .code_stride = code_stride, .width = (uint32_t)width, .tokens = (uint32_t)tokens,
    };
    return launched(lh_launch_q8_rows(LH_Q8_ROWS, &rows, (hipStream_t)stream), "q8 rows");
}

int lh_q8_silu(const float *d_gate, size_t gate_stride, const float *d_up, size_t up_stride,
    size_t width, size_t tokens, int8_t *d_codes, size_t code_stride, float *d_scales,
    void *stream)
{
    if (q8_codes_refused(d_codes, code_stride, d_scales, width, tokens, "q8_silu")) {
        return -1;
    }
    if (!d_gate || !d_up || !aligned(d_gate, 4) || !aligned(d_up, 4) ||
        !stride_ok(gate_stride, width) || !stride_ok(up_stride, width)) {
        return refuse("q8_silu: gate and up in rows of the width required");
    }
    if ((const void *)d_gate == (const void *)d_codes || d_gate == d_scales ||
        (const void *)d_up == (const void *)d_codes || d_up == d_scales) {
        return refuse("q8_silu: codes and scales must not overlap gate or up");
    }
    const lh_q8_source rows = {
        .x = d_gate, .x_stride = gate_stride, .second = d_up, .second_stride = up_stride,
        .scales = d_scales, .codes = d_codes, .code_stride = code_stride,
        .width = (uint32_t)width, .tokens = (uint32_t)tokens,
    };
    return launched(lh_launch_q8_rows(LH_Q8_SILU, &rows, (hipStream_t)stream), "q8 silu");
}

int lh_q8_norm(const float *d_x, size_t x_stride, const float *d_add, size_t add_stride,
    const float *d_gamma, float *d_sum, size_t sum_stride, size_t width, size_t tokens,
    int8_t *d_codes, size_t code_stride, float *d_scales, void *stream)
{
    if (q8_codes_refused(d_codes, code_stride, d_scales, width, tokens, "q8_norm")) {
        return -1;
    }
    if (!d_x || !d_gamma || !aligned(d_x, 4) || !aligned(d_gamma, 4) || !aligned(d_add, 4) ||
        !aligned(d_sum, 4) || !stride_ok(x_stride, width) ||
        (d_add && !stride_ok(add_stride, width)) || (d_sum && !stride_ok(sum_stride, width))) {
        return refuse("q8_norm: x and gamma, and add and sum where given, in rows of the width "
            "required");
    }
    if ((d_sum == d_x && sum_stride != x_stride) ||
        (d_sum && d_sum == d_add && sum_stride != add_stride)) {
        return refuse("q8_norm: a sum in place needs equal strides");
    }
    const void *outputs[] = {d_codes, d_scales, d_sum};
    for (int i = 0; i < 3; i++) {
        if (outputs[i] && (outputs[i] == d_gamma || (i < 2 && (outputs[i] == d_x ||
                outputs[i] == d_add || outputs[i] == d_sum)))) {
            return refuse("q8_norm: codes and scales must not overlap x, add, gamma or the sum, "
                "nor the sum gamma");
        }
    }
    const lh_q8_source rows = {
        .x = d_x, .x_stride = x_stride, .second = d_add, .second_stride = add_stride,
        .gamma = d_gamma, .sum = d_sum, .sum_stride = sum_stride, .scales = d_scales,
        .codes = d_codes, .code_stride = code_stride, .width = (uint32_t)width,
        .tokens = (uint32_t)tokens,
    };
    return launched(lh_launch_q8_rows(LH_Q8_NORM, &rows, (hipStream_t)stream), "q8 norm");
}

static int q8_sizes(size_t rows, size_t cols)
{
    return rows && rows <= ((size_t)1 << 20) && cols && cols <= 65536;
}

size_t lh_q8_bytes(size_t rows, size_t cols)
{
    return q8_sizes(rows, cols) ? (rows + 15) / 16 * ((cols + 127) / 128 * 2048 + 64) : 0;
}

int lh_q8_pack(const int8_t *d_codes, const float *d_scales, size_t rows, size_t cols,
    void *d_packed, void *stream)
{
    if (!d_codes || !d_scales || !d_packed || !q8_sizes(rows, cols) || !aligned(d_packed, 16) ||
        !aligned(d_scales, 4)) {
        return refuse("q8_pack: require pointers (packed on 16 bytes), rows 1..2^20, cols "
            "1..65536");
    }
    return launched(lh_launch_q8_pack(d_codes, d_scales, (uint32_t)rows, (uint32_t)cols, d_packed,
        (hipStream_t)stream), "q8 pack");
}

int lh_q8_quantize(const float *d_w, size_t rows, size_t cols, void *d_packed, void *stream)
{
    if (!d_w || !d_packed || !q8_sizes(rows, cols) || !aligned(d_packed, 16) ||
        !aligned(d_w, 4)) {
        return refuse("q8_quantize: require pointers (packed on 16 bytes), rows 1..2^20, cols "
            "1..65536");
    }
    return launched(lh_launch_q8_quantize(d_w, (uint32_t)rows, (uint32_t)cols, d_packed,
        (hipStream_t)stream), "q8 quantize");
}

size_t lh_q8_scratch(size_t rows, size_t cols, size_t tokens)
{
    if (!q8_sizes(rows, cols) || !tokens || tokens > 65535) {
        return 0;
    }
    return lh_q8_scratch_bytes((uint32_t)rows, (uint32_t)cols, (uint32_t)tokens);
}

int lh_q8_matvec(const void *d_packed, const int8_t *d_x, size_t x_stride,
    const float *d_x_scales, float *d_y, size_t y_stride, size_t rows, size_t cols,
    size_t tokens, void *d_scratch, size_t scratch_bytes, void *stream)
{
    if (q8_codes_refused(d_x, x_stride, d_x_scales, cols, tokens, "q8_matvec")) {
        return -1;
    }
    if (!d_packed || !d_y || !q8_sizes(rows, cols) || !aligned(d_packed, 16) || !aligned(d_y, 4) ||
        !stride_ok(y_stride, rows)) {
        return refuse("q8_matvec: packed weights on 16 bytes, rows 1..2^20 and y in rows of as "
            "many required");
    }
    const size_t need = lh_q8_scratch_bytes((uint32_t)rows, (uint32_t)cols, (uint32_t)tokens);
    if (need && (!d_scratch || scratch_bytes < need || !aligned(d_scratch, 16))) {
        lh_set_error("q8_matvec: needs %zu bytes of scratch on a 16-byte boundary", need);
        return -1;
    }
    if ((const void *)d_x == (const void *)d_y || d_y == d_x_scales ||
        (const void *)d_y == d_packed) {
        return refuse("q8_matvec: y must not overlap x, its scales or the weights");
    }
    return launched(lh_launch_q8_matvec(d_packed, d_x, x_stride, d_x_scales, d_y, y_stride,
        (uint32_t)rows, (uint32_t)cols, (uint32_t)tokens, d_scratch, (hipStream_t)stream),
        "q8 matvec");
}

/* ---- log probabilities ---- */

static int logprobs_sizes(size_t rows, size_t vocab, size_t top)
{
    return rows && rows <= 65535 && vocab && vocab <= ((size_t)1 << 24) &&
        top <= LH_LOGPROBS_TOP;
}

size_t lh_logprobs_scratch(size_t rows, size_t vocab, size_t top)
{
    return logprobs_sizes(rows, vocab, top)
        ? lh_logprobs_scratch_bytes((uint32_t)rows, (uint32_t)vocab, (uint32_t)top) : 0;
}

int lh_logprobs(const float *d_logits, size_t stride, size_t rows, size_t vocab,
    const int64_t *d_tokens, float *d_logprob, float *d_entropy, size_t top, int64_t *d_top_ids,
    float *d_top_logprobs, void *d_scratch, size_t scratch_bytes, void *stream)
{
    if (!d_logits || !logprobs_sizes(rows, vocab, top) || !stride_ok(stride, vocab) ||
        !aligned(d_logits, 4)) {
        return refuse("logprobs: require logits, rows 1..65535, vocab 1..2^24, stride >= vocab, "
            "top 0..64");
    }
    if (!d_tokens != !d_logprob || (top && (!d_top_ids || !d_top_logprobs)) ||
        (!d_logprob && !d_entropy && !top) || !aligned(d_tokens, 8) || !aligned(d_logprob, 4) ||
        !aligned(d_entropy, 4) || !aligned(d_top_ids, 8) || !aligned(d_top_logprobs, 4)) {
        return refuse("logprobs: tokens and logprob go together, top needs ids and "
            "log probabilities, and one output is required");
    }
    const size_t need = lh_logprobs_scratch_bytes((uint32_t)rows, (uint32_t)vocab, (uint32_t)top);
    if (need && (!d_scratch || scratch_bytes < need || !aligned(d_scratch, 16))) {
        lh_set_error("logprobs: needs %zu bytes of scratch on a 16-byte boundary", need);
        return -1;
    }
    return launched(lh_launch_logprobs(d_logits, stride, (uint32_t)rows, (uint32_t)vocab, d_tokens,
        d_logprob, d_entropy, (uint32_t)top, d_top_ids, d_top_logprobs, d_scratch,
        (hipStream_t)stream), "logprobs");
}

/* ---- paged cache ---- */

static int cache_ok(const lh_paged_cache *c)
{
    return c && (c->kind == LH_CACHE_F16 || c->kind == LH_CACHE_Q4) && c->kv_heads &&
        c->kv_heads <= 64 && (c->head_dim == 64 || c->head_dim == 128) && c->page_size &&
        c->page_size <= 1024 && c->page_size % 32 == 0 && c->pages && c->pages <= 0x7fffffffu;
}

size_t lh_paged_cache_bytes(const lh_paged_cache *cache)
{
    if (!cache_ok(cache)) {
        return 0;
    }
    const size_t vector = cache->kind == LH_CACHE_Q4 ? cache->head_dim / 2 + 4
        : (size_t)2 * cache->head_dim;
    return (size_t)cache->pages * cache->kv_heads * cache->page_size * 2 * vector;
}

static int cache_refused(const lh_paged_cache *cache, const char *what)
{
    if (!cache_ok(cache) || !cache->d_pages || !aligned(cache->d_pages, 16)) {
        lh_set_error("%s: cache: kind F16 or Q4, kv_heads 1..64, head_dim 64 or 128, page_size a "
            "multiple of 32 up to 1024, pages 1..2^31-1 on a 16-byte boundary required", what);
        return 1;
    }
    return 0;
}

static int batch_ok(const lh_paged_batch *b)
{
    return b && b->sequences && b->sequences <= 65535 && b->tokens && b->tokens <= (1u << 24) &&
        b->table_width && b->table_width <= (1u << 20) && b->max_query && b->max_length;
}

static int batch_refused(const lh_paged_batch *b, const char *what)
{
    if (!batch_ok(b) || !b->d_query_start || !b->d_length || !b->d_table ||
        !aligned(b->d_query_start, 4) || !aligned(b->d_length, 4) || !aligned(b->d_table, 4)) {
        lh_set_error("%s: batch: sequences 1..65535, tokens 1..2^24, table_width 1..2^20, "
            "max_query, max_length and the three arrays required", what);
        return 1;
    }
    return 0;
}

static int heads_ok(uint32_t heads, uint32_t kv_heads)
{
    return heads && heads % kv_heads == 0 && heads / kv_heads <= 64;
}

int lh_paged_append(const lh_paged_cache *cache, const lh_paged_batch *batch, uint32_t heads,
    const float *d_q, size_t q_stride, const float *d_k, size_t k_stride, const float *d_v,
    size_t v_stride, const float *d_cos, const float *d_sin, uint32_t positions,
    const float *d_qfactor, float *d_q_out, size_t q_out_stride, void *stream)
{
    if (cache_refused(cache, "paged_append") || batch_refused(batch, "paged_append")) {
        return -1;
    }
    const size_t kv = (size_t)cache->kv_heads * cache->head_dim;
    const size_t q = (size_t)heads * cache->head_dim;
    if (!d_k || !d_v || !stride_ok(k_stride, kv) || !stride_ok(v_stride, kv) ||
        !aligned(d_k, 4) || !aligned(d_v, 4)) {
        return refuse("paged_append: keys and values with rows of kv_heads * head_dim required");
    }
    if (heads && (!heads_ok(heads, cache->kv_heads) || !d_q || !d_q_out ||
            !stride_ok(q_stride, q) || !stride_ok(q_out_stride, q) || !aligned(d_q, 4) ||
            !aligned(d_q_out, 4))) {
        return refuse("paged_append: heads a multiple of kv_heads, up to 64 times, with queries "
            "and their output in rows of heads * head_dim required (or heads 0)");
    }
    if (heads && d_q == d_q_out && q_stride != q_out_stride) {
        return refuse("paged_append: queries in place need equal strides");
    }
    if (!d_cos != !d_sin || ((d_cos || (heads && d_qfactor)) && !positions) ||
        !aligned(d_cos, 4) || !aligned(d_sin, 4) || !aligned(d_qfactor, 4)) {
        return refuse("paged_append: cos and sin go together, and they and qfactor have one or "
            "more positions");
    }
    const lh_append_rows rows = {
        .q = d_q, .k = d_k, .v = d_v, .cosine = d_cos, .sine = d_sin,
        .qfactor = heads ? d_qfactor : NULL, .q_out = d_q_out, .q_stride = q_stride,
        .k_stride = k_stride, .v_stride = v_stride, .q_out_stride = q_out_stride,
        .group = heads / cache->kv_heads, .positions = positions,
    };
    return launched(lh_launch_paged_append(cache, batch, &rows, (hipStream_t)stream),
        "paged append");
}

int lh_paged_read(const lh_paged_cache *cache, const lh_paged_batch *batch, float *d_keys,
    size_t k_stride, float *d_values, size_t v_stride, void *stream)
{
    if (cache_refused(cache, "paged_read") || batch_refused(batch, "paged_read")) {
        return -1;
    }
    const size_t kv = (size_t)cache->kv_heads * cache->head_dim;
    if ((!d_keys && !d_values) || (d_keys && !stride_ok(k_stride, kv)) ||
        (d_values && !stride_ok(v_stride, kv)) || !aligned(d_keys, 4) || !aligned(d_values, 4)) {
        return refuse("paged_read: keys or values with rows of kv_heads * head_dim required");
    }
    return launched(lh_launch_paged_read(cache, batch, d_keys, k_stride, d_values, v_stride,
        (hipStream_t)stream), "paged read");
}

size_t lh_paged_attention_scratch(const lh_paged_cache *cache, const lh_paged_batch *batch,
    uint32_t heads)
{
    if (!cache_ok(cache) || !batch_ok(batch) || !heads_ok(heads, cache->kv_heads)) {
        return 0;
    }
    return lh_paged_attention_scratch_bytes(cache, batch, heads / cache->kv_heads);
}

int lh_paged_attention(const lh_paged_cache *cache, const lh_paged_batch *batch, uint32_t heads,
    const float *d_q, size_t q_stride, float scale, float *d_out, size_t out_stride,
    void *d_scratch, size_t scratch_bytes, void *stream)
{
    if (cache_refused(cache, "paged_attention") || batch_refused(batch, "paged_attention")) {
        return -1;
    }
    const size_t q = (size_t)heads * cache->head_dim;
    if (!heads_ok(heads, cache->kv_heads) || !d_q || !d_out || d_q == d_out ||
        !stride_ok(q_stride, q) || !stride_ok(out_stride, q) || !aligned(d_q, 4) ||
        !aligned(d_out, 4)) {
        return refuse("paged_attention: heads a multiple of kv_heads, up to 64 times, with "
            "queries and another output in rows of heads * head_dim required");
    }
    if (!(scale > 0) || !isfinite(scale)) {
        return refuse("paged_attention: scale must be positive and finite");
    }
    const size_t need = lh_paged_attention_scratch_bytes(cache, batch, heads / cache->kv_heads);
    if (need && (!d_scratch || scratch_bytes < need || !aligned(d_scratch, 16))) {
        lh_set_error("paged_attention: needs %zu bytes of scratch on a 16-byte boundary", need);
        return -1;
    }
    return launched(lh_launch_paged_attention(cache, batch, heads / cache->kv_heads, d_q, q_stride,
        scale, d_out, out_stride, d_scratch, (hipStream_t)stream), "paged attention");
}

/* ---- beam search ---- */

static int beam_sizes(size_t groups, size_t beams, size_t vocab, size_t keep)
{
    return groups && groups <= 65535 && beams && beams <= LH_BEAMS && groups * beams <= 65535 &&
        vocab && vocab <= ((size_t)1 << 24) && keep && keep <= LH_BEAMS;
}

size_t lh_beam_scratch(size_t groups, size_t beams, size_t vocab, size_t keep)
{
    return beam_sizes(groups, beams, vocab, keep) ? lh_beam_scratch_bytes((uint32_t)groups,
        (uint32_t)beams, (uint32_t)vocab, (uint32_t)keep) : 0;
}

int lh_beam_select(const float *d_logits, size_t stride, size_t groups, size_t beams,
    size_t vocab, const float *d_scores, const uint8_t *d_done, int64_t stop, size_t keep,
    int32_t *d_parent, int64_t *d_token, float *d_score, uint8_t *d_done_out, void *d_scratch,
    size_t scratch_bytes, void *stream)
{
    if (!d_logits || !d_scores || !beam_sizes(groups, beams, vocab, keep) ||
        !stride_ok(stride, vocab) || !aligned(d_logits, 4) || !aligned(d_scores, 4)) {
        return refuse("beam_select: require logits and scores, groups * beams 1..65535, beams and "
            "keep 1..64, vocab 1..2^24, stride >= vocab");
    }
    if (!d_parent || !d_token || !d_score || !aligned(d_parent, 4) || !aligned(d_token, 8) ||
        !aligned(d_score, 4)) {
        return refuse("beam_select: parents, tokens and scores of the kept places required");
    }
    if (d_score == d_scores || (d_done && d_done == d_done_out)) {
        return refuse("beam_select: outputs must not overlap inputs");
    }
    const size_t need = lh_beam_scratch(groups, beams, vocab, keep);
    if (need && (!d_scratch || scratch_bytes < need || !aligned(d_scratch, 16))) {
        lh_set_error("beam_select: needs %zu bytes of scratch on a 16-byte boundary", need);
        return -1;
    }
    const lh_beam_choice choice = {
        .logits = d_logits, .scores = d_scores, .done = d_done, .parent = d_parent,
        .token = d_token, .stop = stop, .score = d_score, .done_out = d_done_out,
        .stride = stride, .groups = (uint32_t)groups, .beams = (uint32_t)beams,
        .vocab = (uint32_t)vocab, .keep = (uint32_t)keep,
    };
    return launched(lh_launch_beam_select(&choice, d_scratch, (hipStream_t)stream),
        "beam select");
}

int lh_beam_reorder(const lh_paged_cache *caches, size_t layers, size_t groups, size_t beams,
    const int32_t *d_parent, const int32_t *d_length, const int32_t *d_table,
    int32_t *d_table_out, size_t table_width, void *stream)
{
    if (!caches || !layers || layers > LH_BEAM_LAYERS) {
        return refuse("beam_reorder: 1..64 layers of caches required");
    }
    for (size_t i = 0; i < layers; i++) {
        const lh_paged_cache *c = &caches[i];
        if (cache_refused(c, "beam_reorder")) {
            return -1;
        }
        if (c->kind != caches->kind || c->kv_heads != caches->kv_heads ||
            c->head_dim != caches->head_dim || c->page_size != caches->page_size ||
            c->pages != caches->pages) {
            return refuse("beam_reorder: the caches of all layers must be alike");
        }
    }
    if (!groups || groups > 65535 || !beams || beams > LH_BEAMS || groups * beams > 65535 ||
        !table_width || table_width > ((size_t)1 << 20) || !d_parent || !d_length || !d_table ||
        !d_table_out || !aligned(d_parent, 4) || !aligned(d_length, 4) || !aligned(d_table, 4) ||
        !aligned(d_table_out, 4)) {
        return refuse("beam_reorder: require parents, lengths and tables, groups * beams 1..65535, "
            "beams 1..64, table_width 1..2^20");
    }
    if (d_table_out == d_parent || d_table_out == d_length) {
        return refuse("beam_reorder: the tables must not overlap parents or lengths");
    }
    return launched(lh_launch_beam_reorder(caches, (uint32_t)layers, (uint32_t)groups,
        (uint32_t)beams, d_parent, d_length, d_table, d_table_out, (uint32_t)table_width,
        (hipStream_t)stream), "beam reorder");
}
