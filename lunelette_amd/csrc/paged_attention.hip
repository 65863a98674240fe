// Causal attention over the paged KV cache (lh_paged_attention).
#include "lh_paged.h"

namespace lh {

template <int D, bool Q4>
__device__ __forceinline__ float key_at(const uint8_t* part, uint32_t page_size, uint32_t slot,
    uint32_t d)
{
    typedef PageLayout<D, Q4> Layout;
    const uint8_t* at = part + Layout::key_chunk(slot, d >> 3);
    if (!Q4) {
        return (float)reinterpret_cast<const _Float16*>(at)[d & 7];
    }
    const uint32_t w = *reinterpret_cast<const uint32_t*>(part + Layout::scales(page_size, 0) +
        4 * slot);
    return __builtin_fmaf((float)(*reinterpret_cast<const uint32_t*>(at) >> nibble_at(d & 7) & 15u),
        bf16_to_f32(w & 0xffffu), bf16_to_f32(w >> 16));
}

template <int D, bool Q4>
__device__ __forceinline__ float value_at(const uint8_t* part, uint32_t page_size, uint32_t slot,
    uint32_t d)
{
    typedef PageLayout<D, Q4> Layout;
    const uint8_t* at = part + Layout::values(page_size) +
        Layout::value_chunk(slot, d, (slot >> 2) & 3);
    const uint32_t e = (slot & 3) + 4 * ((slot >> 4) & 1);
    if (!Q4) {
        return (float)reinterpret_cast<const _Float16*>(at)[e];
    }
    const uint32_t w = *reinterpret_cast<const uint32_t*>(part + Layout::scales(page_size, 1) +
        4 * slot);
    return __builtin_fmaf((float)(*reinterpret_cast<const uint32_t*>(at) >> nibble_at(e) & 15u),
        bf16_to_f32(w & 0xffffu), bf16_to_f32(w >> 16));
}

// One wave a (token, head): positions one after another with the running maximum
// and sum of the softmax, a lane the dims l and l + 64.
template <int D, bool Q4>
__global__ void __launch_bounds__(64)
k_paged_attention(Pages cache, Batch batch, uint32_t group, const float* __restrict__ q,
    size_t q_stride, float scale, float* __restrict__ out, size_t out_stride)
{
    constexpr int N = D / 64;
    const uint32_t head = blockIdx.y, s = blockIdx.z, lane = threadIdx.x;
    const Span span = batch_span(batch, s);
    for (int64_t t = blockIdx.x; t < span.count; t += gridDim.x) {
        const size_t row = (size_t)(span.begin + t);
        float qd[N], acc[N] = {}, m = -__builtin_inff(), sum = 0;
        for (int n = 0; n < N; n++) {
            qd[n] = q[row * q_stride + head * D + lane + 64 * n];
        }
        const int64_t last = span.first + t;
        bool lost = last >= (int64_t)batch.width * cache.page_size;
        for (int64_t p = 0; p <= last && !lost; p++) {
            const uint8_t* part = page_part<D, Q4>(cache, batch, s, p, head / group);
            if (!part) {
                lost = true;
                break;
            }
            const uint32_t slot = (uint32_t)(p % cache.page_size);
            float dot = 0;
            for (int n = 0; n < N; n++) {
                dot = __builtin_fmaf(qd[n],
                    key_at<D, Q4>(part, cache.page_size, slot, lane + 64 * n), dot);
            }
            const float score = wave_lane0(wave_tree64(dot)) * scale;
            const float top = fmaxf(m, score), shift = top > -__builtin_inff() ? top : 0.0f;
            const float keep = expf_cw(m - shift), e = expf_cw(score - shift);
            m = top;
            sum = __builtin_fmaf(sum, keep, e);
            for (int n = 0; n < N; n++) {
                acc[n] = __builtin_fmaf(e,
                    value_at<D, Q4>(part, cache.page_size, slot, lane + 64 * n), acc[n] * keep);
            }
        }
        for (int n = 0; n < N; n++) {
            out[row * out_stride + head * D + lane + 64 * n] =
                lost ? __builtin_nanf("") : last < 0 ? 0.0f : acc[n] / sum;
        }
    }
}

}  // namespace lh

using namespace lh;

extern "C" size_t lh_paged_attention_scratch_bytes(const lh_paged_cache* cache,
    const lh_paged_batch* batch, uint32_t group)
{
    (void)cache;
    (void)batch;
    (void)group;
    return 0;
}

template <int D, bool Q4>
static void attention(const lh_paged_cache* c, const lh_paged_batch* b, uint32_t group,
    const float* q, size_t q_stride, float scale, float* out, size_t out_stride, hipStream_t s)
{
    const uint32_t query = b->max_query < b->tokens ? b->max_query : b->tokens;
    hipLaunchKernelGGL((k_paged_attention<D, Q4>), dim3(query, c->kv_heads * group, b->sequences),
        dim3(64), 0, s, pages_of(c), batch_of(b), group, q, q_stride, scale, out, out_stride);
}

extern "C" int lh_launch_paged_attention(const lh_paged_cache* cache, const lh_paged_batch* batch,
    uint32_t group, const float* q, size_t q_stride, float scale, float* out, size_t out_stride,
    uint8_t* scratch, hipStream_t s)
{
    (void)scratch;
    LH_FOR_CACHE(cache, attention, cache, batch, group, q, q_stride, scale, out, out_stride, s);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
