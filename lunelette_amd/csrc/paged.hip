// The paged KV cache: append with rotation, reading back (lh_paged_append,
// lh_paged_read).
#include "lh_paged.h"

namespace lh {

__device__ __forceinline__ double wave_min(double v)
{
    for (int s = 32; s; s >>= 1) {
        v = fmin(v, __shfl_xor(v, s));
    }
    return v;
}

__device__ __forceinline__ double wave_max(double v)
{
    for (int s = 32; s; s >>= 1) {
        v = fmax(v, __shfl_xor(v, s));
    }
    return v;
}

// Scale (low half) and zero (high half) of a vector whose lanes hold a and b
// (lanes with on = false hold nothing). 64-bit differences and quotients: the
// codes are those of the exact rotation unless a value lies within 2^-50 of a
// border.
__device__ __forceinline__ uint32_t q4_word(double a, double b, bool on)
{
    const bool finite = !on || (__builtin_isfinite(a) && __builtin_isfinite(b));
    const double low = wave_min(on ? fmin(a, b) : __builtin_inf());
    const double high = wave_max(on ? fmax(a, b) : -__builtin_inf());
    const uint32_t z = bf16_nearest((float)low);
    const float zero = bf16_to_f32(z);
    const float step = (float)((high - (double)zero) / 15.0);
    const uint32_t s = step > 0 ? bf16_nearest(step) : 0;
    if (__ballot(!finite) || !__builtin_isfinite(zero) || !__builtin_isfinite(bf16_to_f32(s))) {
        return 0x7fc07fc0u;
    }
    return s | z << 16;
}

__device__ __forceinline__ uint32_t q4_code(double v, uint32_t word)
{
    const float s = bf16_to_f32(word & 0xffffu), z = bf16_to_f32(word >> 16);
    if (!(s > 0)) {
        return 0;
    }
    return (uint32_t)fmin(fmax(rint((v - (double)z) / (double)s), 0.0), 15.0);
}

// A workgroup takes the tokens of one sequence in one 32-position block, for one KV
// head: no other workgroup writes that part of a page, so the words that hold
// several positions' values are merged without atomics. Waves take vectors (key,
// value, the KV head's queries of each token), a lane the dims l and l + D / 2 of one;
// keys and values meet in LDS and leave in the page's order.
template <int D, bool Q4>
__global__ void __launch_bounds__(512)
k_paged_append(Pages cache, Batch batch, lh_append_rows rows)
{
    typedef PageLayout<D, Q4> Layout;
    constexpr int H = D / 2;
    __shared__ uint8_t codes[2][32][Q4 ? D : 1];
    __shared__ _Float16 halves[2][32][Q4 ? 1 : D];
    const uint32_t h = blockIdx.y, s = blockIdx.z;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Span span = batch_span(batch, s);
    if (!span.count) {
        return;
    }
    const int64_t block0 = span.first >> 5;
    const int64_t blocks = ((span.first + span.count - 1) >> 5) - block0 + 1;
    const bool on = lane < H;
    const uint32_t l = on ? lane : 0;
    for (int64_t u = blockIdx.x; u < blocks; u += gridDim.x) {
        const int64_t base = 32 * (block0 + u);
        const int64_t p0 = base > span.first ? base : span.first;
        const int64_t end = span.first + span.count;
        const int64_t p1 = base + 32 < end ? base + 32 : end;
        uint8_t* part = page_part<D, Q4>(cache, batch, s, base, h);
        const uint32_t slot0 = part ? (uint32_t)(base % cache.page_size) : 0;
        const uint32_t vectors = (uint32_t)(p1 - p0) * (2 + rows.group);
        __syncthreads();
        for (uint32_t i = wave; i < vectors; i += 8) {
            const uint32_t which = i % (2 + rows.group);
            const int64_t p = p0 + i / (2 + rows.group);
            const size_t token = (size_t)(span.begin + (p - span.first));
            const bool turned = rows.cosine && which != 1;
            const bool placed = p >= 0 && (!(rows.cosine || rows.qfactor) || p < rows.positions);
            const uint32_t head = which < 2 ? h : h * rows.group + which - 2;
            const float* x = which == 0 ? rows.k + token * rows.k_stride
                : which == 1 ? rows.v + token * rows.v_stride : rows.q + token * rows.q_stride;
            x += (size_t)head * D;
            double a = x[l], b = x[l + H];
            if (turned && placed) {
                const float* c = rows.cosine + (size_t)p * D;
                const float* n = rows.sine + (size_t)p * D;
                const double ra = a * (double)c[l] - b * (double)n[l];
                b = b * (double)c[l + H] + a * (double)n[l + H];
                a = ra;
            }
            if (which >= 2) {
                const double f = rows.qfactor && placed ? (double)rows.qfactor[p] : 1.0;
                float* out = rows.q_out + token * rows.q_out_stride + (size_t)head * D;
                const float nan = __builtin_nanf("");
                if (on) {
                    out[l] = placed ? (float)(a * f) : nan;
                    out[l + H] = placed ? (float)(b * f) : nan;
                }
                continue;
            }
            const uint32_t at = (uint32_t)(p - base);
            if (Q4) {
                const uint32_t word = q4_word(a, b, on);
                if (on) {
                    codes[which][at][l] = (uint8_t)q4_code(a, word);
                    codes[which][at][l + H] = (uint8_t)q4_code(b, word);
                }
                if (part && placed && lane == 0) {
                    *reinterpret_cast<uint32_t*>(part +
                        Layout::scales(cache.page_size, which) + 4 * (slot0 + at)) = word;
                }
            } else if (on) {
                halves[which][at][l] = (_Float16)(float)a;
                halves[which][at][l + H] = (_Float16)(float)b;
            }
        }
        __syncthreads();
        if (!part) {
            continue;
        }
        // Slots of the block that are written: [from, to).
        const int64_t bound = rows.cosine || rows.qfactor ? rows.positions : p1;
        const uint32_t from = (uint32_t)(p0 - base);
        const uint32_t to = (uint32_t)((p1 < bound ? p1 : bound > p0 ? bound : p0) - base);
        for (uint32_t i = threadIdx.x; i < (to - from) * (D / 8); i += 512) {
            const uint32_t at = from + i / (D / 8), c = i % (D / 8);
            uint8_t* out = part + Layout::key_chunk(slot0 + at, c);
            if (Q4) {
                uint32_t word = 0;
                for (int e = 0; e < 8; e++) {
                    word |= (uint32_t)codes[0][at][8 * c + e] << nibble_at(e);
                }
                *reinterpret_cast<uint32_t*>(out) = word;
            } else {
                *reinterpret_cast<uint4*>(out) = *reinterpret_cast<uint4*>(&halves[0][at][8 * c]);
            }
        }
        for (uint32_t i = threadIdx.x; i < 4 * D && to > from; i += 512) {
            const uint32_t d = i % D, g = i / D;
            uint8_t* out = part + Layout::values(cache.page_size) +
                Layout::value_chunk(slot0, d, g);
            uint32_t word = 0, mask = 0;
            for (int e = 0; e < 8; e++) {
                const uint32_t at = 4 * g + (e & 3) + 16 * (e >> 2);
                if (at < from || at >= to) {
                    continue;
                }
                if (Q4) {
                    word |= (uint32_t)codes[1][at][d] << nibble_at(e);
                    mask |= 15u << nibble_at(e);
                } else {
                    reinterpret_cast<_Float16*>(out)[e] = halves[1][at][d];
                }
            }
            if (Q4 && mask) {
                uint32_t* w = reinterpret_cast<uint32_t*>(out);
                *w = mask == ~0u ? word : (*w & ~mask) | word;
            }
        }
    }
}

// One FP32 element a thread and step: grid (units, KV heads, sequences).
template <int D, bool Q4>
__global__ void __launch_bounds__(256)
k_paged_read(Pages cache, Batch batch, float* __restrict__ keys, size_t k_stride,
    float* __restrict__ values, size_t v_stride)
{
    typedef PageLayout<D, Q4> Layout;
    const uint32_t h = blockIdx.y, s = blockIdx.z;
    const Span span = batch_span(batch, s);
    const uint32_t d = threadIdx.x % D, step = 256 / D;
    for (int64_t t = (int64_t)blockIdx.x * step + threadIdx.x / D; t < span.count;
         t += (int64_t)gridDim.x * step) {
        const int64_t p = span.first + t;
        const uint8_t* part = page_part<D, Q4>(cache, batch, s, p, h);
        const uint32_t slot = part ? (uint32_t)(p % cache.page_size) : 0;
        const uint32_t e = (slot & 3) + 4 * ((slot >> 4) & 1);
        for (int which = 0; which < 2; which++) {
            float* out = which ? values : keys;
            if (!out) {
                continue;
            }
            float v = __builtin_nanf("");
            if (part) {
                const uint8_t* at = which ? part + Layout::values(cache.page_size) +
                        Layout::value_chunk(slot, d, (slot >> 2) & 3)
                    : part + Layout::key_chunk(slot, d >> 3);
                const uint32_t element = which ? e : d & 7;
                if (Q4) {
                    const uint32_t code = *reinterpret_cast<const uint32_t*>(at) >>
                        nibble_at(element) & 15u;
                    const uint32_t word = *reinterpret_cast<const uint32_t*>(part +
                        Layout::scales(cache.page_size, which) + 4 * slot);
                    v = __builtin_fmaf((float)code, bf16_to_f32(word & 0xffffu),
                        bf16_to_f32(word >> 16));
                } else {
                    v = (float)reinterpret_cast<const _Float16*>(at)[element];
                }
            }
            out[(size_t)(span.begin + t) * (which ? v_stride : k_stride) + (size_t)h * D + d] = v;
        }
    }
}

}  // namespace lh

using namespace lh;

template <int D, bool Q4>
static void append(const lh_paged_cache* c, const lh_paged_batch* b, const lh_append_rows* rows,
    hipStream_t s)
{
    const uint32_t query = b->max_query < b->tokens ? b->max_query : b->tokens;
    const uint32_t blocks = (query + 30) / 32 + 1;
    hipLaunchKernelGGL((k_paged_append<D, Q4>), dim3(blocks, c->kv_heads, b->sequences), dim3(512),
        0, s, pages_of(c), batch_of(b), *rows);
}

template <int D, bool Q4>
static void read(const lh_paged_cache* c, const lh_paged_batch* b, float* keys, size_t k_stride,
    float* values, size_t v_stride, hipStream_t s)
{
    const uint32_t query = b->max_query < b->tokens ? b->max_query : b->tokens;
    const uint32_t step = 256 / D;
    hipLaunchKernelGGL((k_paged_read<D, Q4>), dim3((query + step - 1) / step, c->kv_heads,
        b->sequences), dim3(256), 0, s, pages_of(c), batch_of(b), keys, k_stride, values, v_stride);
}

extern "C" int lh_launch_paged_append(const lh_paged_cache* cache, const lh_paged_batch* batch,
    const lh_append_rows* rows, hipStream_t s)
{
    LH_FOR_CACHE(cache, append, cache, batch, rows, s);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

extern "C" int lh_launch_paged_read(const lh_paged_cache* cache, const lh_paged_batch* batch,
    float* keys, size_t k_stride, float* values, size_t v_stride, hipStream_t s)
{
    LH_FOR_CACHE(cache, read, cache, batch, keys, k_stride, values, v_stride, s);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
