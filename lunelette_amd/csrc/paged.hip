// The paged KV cache: append with rotation, reading back (lh_paged_append,
// lh_paged_read). Both are memory round trips: a workgroup takes the tokens of one
// sequence in one 32-position block of a page for one KV head, asks for everything at
// once, and goes through LDS into the other order.
#include "lh_mfma.h"
#include "lh_paged.h"

namespace lh {

// Lane l's word of lane l + N (mod 16) of its 16.
template <int N>
__device__ __forceinline__ uint32_t row_turn(uint32_t v)
{
    return __builtin_amdgcn_mov_dpp(v, 0x120 + N, 0xf, 0xf, false);   // row_ror
}

template <int N>
__device__ __forceinline__ double row_turn(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)row_turn<N>((uint32_t)(u >> 32)) << 32 |
        row_turn<N>((uint32_t)u));
}

// Over 16 lanes, in each of them.
__device__ __forceinline__ double row_max(double v)
{
    v = fmax(v, row_turn<8>(v));
    v = fmax(v, row_turn<4>(v));
    v = fmax(v, row_turn<2>(v));
    return fmax(v, row_turn<1>(v));
}

// Scale (low half) and zero (high half) of a vector of which 16 lanes hold N values
// each. 64-bit differences and quotients: the codes are those of the exact rotation
// unless a value lies within 2^-50 of a border.
template <int N>
__device__ __forceinline__ uint32_t q4_word(const double (&v)[N], uint32_t lane)
{
    bool finite = true;
    double low = v[0], high = v[0];
#pragma unroll
    for (int i = 0; i < N; i++) {
        finite &= __builtin_isfinite(v[i]);
        low = fmin(low, v[i]);
        high = fmax(high, v[i]);
    }
    low = -row_max(-low);
    high = row_max(high);
    const uint32_t z = bf16_nearest((float)low);
    const float zero = bf16_to_f32(z);
    const float step = (float)((high - (double)zero) / 15.0);
    const uint32_t s = step > 0 ? bf16_nearest(step) : 0;
    const bool odd = (__ballot(!finite) >> (lane & 48) & 0xffffu) != 0;
    if (odd || !__builtin_isfinite(zero) || !__builtin_isfinite(bf16_to_f32(s))) {
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

// N floats (2 or 4) from and to any 4-byte boundary.
template <int N>
struct Few {
    typedef float any __attribute__((ext_vector_type(N), aligned(4)));

    __device__ __forceinline__ static void load(const float* p, double* to)
    {
        const any v = *reinterpret_cast<const any*>(p);
#pragma unroll
        for (int i = 0; i < N; i++) {
            to[i] = v[i];
        }
    }
    __device__ __forceinline__ static void store(float* p, const double* from, float nan)
    {
        any v;
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i] = (float)from[i] + nan;
        }
        *reinterpret_cast<any*>(p) = v;
    }
};

// A lane's dims of a vector, N / 2 from dim `at` and as many from D / 2 + at, turned by
// the rows of position p: formed in 64 bits.
template <int D, int N>
__device__ __forceinline__ void rotate(double (&v)[N], const lh_append_rows& rows, int64_t p,
    uint32_t at)
{
    constexpr int H = N / 2;
    double c[N], s[N];
    const float *cosine = rows.cosine + (size_t)p * D + at, *sine = rows.sine + (size_t)p * D + at;
    Few<H>::load(cosine, c);
    Few<H>::load(cosine + D / 2, c + H);
    Few<H>::load(sine, s);
    Few<H>::load(sine + D / 2, s + H);
#pragma unroll
    for (int i = 0; i < H; i++) {
        const double a = v[i] * c[i] - v[H + i] * s[i];
        v[H + i] = v[H + i] * c[H + i] + v[i] * s[H + i];
        v[i] = a;
    }
}

// The tokens of a sequence in one 32-position block: positions from .. to - 1 of it.
struct Unit {
    int64_t base, first;   // positions of the block and of its first token
    size_t token;          // that token's row
    uint32_t from, to;
};

__device__ __forceinline__ Unit unit_of(const Span& span, int64_t u)
{
    const int64_t base = 32 * ((span.first >> 5) + u), end = span.first + span.count;
    const int64_t first = base > span.first ? base : span.first;
    return {base, first, (size_t)(span.begin + (first - span.first)), (uint32_t)(first - base),
        (uint32_t)((base + 32 < end ? base + 32 : end) - base)};
}

__device__ __forceinline__ int64_t units_of(const Span& span)
{
    return span.count ? ((span.first + span.count - 1) >> 5) - (span.first >> 5) + 1 : 0;
}

// grid (units, KV heads twice, sequences): a KV head's keys and values, then its
// queries. No other workgroup writes the unit's part of the page, so the words that
// hold several positions' values are merged without atomics. Sixteen lanes take a
// vector.
template <int D, bool Q4>
__global__ void __launch_bounds__(256)
k_paged_append(Pages cache, Batch batch, lh_append_rows rows)
{
    typedef PageLayout<D, Q4> Layout;
    constexpr int N = D / 16, H = N / 2, WORDS = 4 * D / 256;
    __shared__ uint8_t codes[2][32][Q4 ? D : 1];
    __shared__ _Float16 halves[2][32][Q4 ? 1 : D];
    const bool queries = blockIdx.y >= cache.kv_heads;
    const uint32_t h = queries ? blockIdx.y - cache.kv_heads : blockIdx.y, s = blockIdx.z;
    const uint32_t lane = threadIdx.x & 63;
    const Span span = batch_span(batch, s);
    const int64_t units = units_of(span);
    const bool bounded = rows.cosine || rows.qfactor;   // by the rotation's rows
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const Unit unit = unit_of(span, u);
        const uint32_t count = unit.to - unit.from;
        if (queries) {
            const uint32_t each = rows.group * (D / N);   // lanes of a token's queries
            for (uint32_t i = threadIdx.x; i < count * each; i += 256) {
                const uint32_t t = i / each, rest = i % each, at = (rest % (D / N)) * H;
                const int64_t p = unit.first + t;
                const size_t head = (size_t)h * rows.group + rest / (D / N);
                const float* x = rows.q + (unit.token + t) * rows.q_stride + head * D + at;
                double v[N];
                Few<H>::load(x, v);
                Few<H>::load(x + D / 2, v + H);
                const bool placed = p >= 0 && (!bounded || p < rows.positions);
                if (placed && rows.cosine) {
                    rotate<D>(v, rows, p, at);
                }
                if (placed && rows.qfactor) {
                    const double f = rows.qfactor[p];
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        v[e] *= f;
                    }
                }
                float* out = rows.q_out + (unit.token + t) * rows.q_out_stride + head * D + at;
                const float nan = placed ? 0.0f : __builtin_nanf("");
                Few<H>::store(out, v, nan);
                Few<H>::store(out + D / 2, v + H, nan);
            }
            continue;
        }
        uint8_t* part = page_part<D, Q4>(cache, batch, s, unit.base, h);
        const uint32_t slot0 = part ? (uint32_t)(unit.base % cache.page_size) : 0;
        // Slots that are written: [from, to).
        const int64_t bound = bounded ? rows.positions - unit.base : 32;
        const uint32_t from = unit.from;
        const uint32_t to = bound < from ? from : bound < unit.to ? (uint32_t)bound : unit.to;
        // Words that keep other positions' values: asked for now.
        uint32_t* word[WORDS];
        uint32_t old[WORDS], mask[WORDS];
        if (Q4) {
#pragma unroll
            for (int w = 0; w < WORDS; w++) {
                const uint32_t i = threadIdx.x + 256 * w, d = i % D, g = i / D;
                mask[w] = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t at = 4 * g + (e & 3) + 16 * (e >> 2);
                    mask[w] |= at >= from && at < to ? 15u << nibble_at(e) : 0;
                }
                if (!part) {
                    mask[w] = 0;
                    continue;
                }
                word[w] = reinterpret_cast<uint32_t*>(part + Layout::values(cache.page_size) +
                    Layout::value_chunk(slot0, d, g));
                old[w] = mask[w] && mask[w] != ~0u ? *word[w] : 0;
            }
        }
        if (u != blockIdx.x) {
            __syncthreads();   // the previous unit's readers
        }
        for (uint32_t i = threadIdx.x >> 4; i < 2 * count; i += 16) {
            const uint32_t which = i & 1, t = i >> 1, at = (threadIdx.x & 15) * H;
            const int64_t p = unit.first + t;
            const float* x = (which ? rows.v + (unit.token + t) * rows.v_stride
                : rows.k + (unit.token + t) * rows.k_stride) + (size_t)h * D + at;
            double v[N];
            Few<H>::load(x, v);
            Few<H>::load(x + D / 2, v + H);
            if (!which && rows.cosine && p >= 0 && p < rows.positions) {
                rotate<D>(v, rows, p, at);
            }
            const uint32_t slot = from + t;
            if (Q4) {
                const uint32_t scale = q4_word(v, lane);
#pragma unroll
                for (int e = 0; e < N; e++) {
                    codes[which][slot][at + (e % H) + (e / H) * (D / 2)] =
                        (uint8_t)q4_code(v[e], scale);
                }
                if (part && slot < to && at == 0) {
                    *reinterpret_cast<uint32_t*>(part +
                        Layout::scales(cache.page_size, which) + 4 * (slot0 + slot)) = scale;
                }
            } else {
#pragma unroll
                for (int e = 0; e < N; e++) {
                    halves[which][slot][at + (e % H) + (e / H) * (D / 2)] = (_Float16)(float)v[e];
                }
            }
        }
        __syncthreads();
        if (!part) {
            continue;
        }
        for (uint32_t i = threadIdx.x; i < (to - from) * (D / 8); i += 256) {
            const uint32_t at = from + i / (D / 8), c = i % (D / 8);
            uint8_t* out = part + Layout::key_chunk(slot0 + at, c);
            if (Q4) {
                uint32_t x = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    x |= (uint32_t)codes[0][at][8 * c + e] << nibble_at(e);
                }
                *reinterpret_cast<uint32_t*>(out) = x;
            } else {
                *reinterpret_cast<uint4*>(out) = *reinterpret_cast<uint4*>(&halves[0][at][8 * c]);
            }
        }
#pragma unroll
        for (int w = 0; w < WORDS; w++) {
            const uint32_t i = threadIdx.x + 256 * w, d = i % D, g = i / D;
            if (Q4) {
                uint32_t x = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    // (Slots without a token hold anything.)
                    x |= (codes[1][4 * g + (e & 3) + 16 * (e >> 2)][d] & 15u) << nibble_at(e);
                }
                if (mask[w]) {
                    *word[w] = (x & mask[w]) | (old[w] & ~mask[w]);
                }
                continue;
            }
            _Float16* out = reinterpret_cast<_Float16*>(part + Layout::values(cache.page_size) +
                Layout::value_chunk(slot0, d, g));
            f16x8 x;
            uint32_t present = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t at = 4 * g + (e & 3) + 16 * (e >> 2);
                x[e] = halves[1][at][d];
                present |= at >= from && at < to ? 1u << e : 0;
            }
            if (present == 0xffu) {
                *reinterpret_cast<f16x8*>(out) = x;
                continue;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (present >> e & 1) {
                    out[e] = x[e];
                }
            }
        }
    }
}

// grid (units, KV heads, sequences).
template <int D, bool Q4>
__global__ void __launch_bounds__(256)
k_paged_read(Pages cache, Batch batch, float* __restrict__ keys, size_t k_stride,
    float* __restrict__ values, size_t v_stride)
{
    typedef PageLayout<D, Q4> Layout;
    __shared__ float rows[32][D + 1];
    const uint32_t h = blockIdx.y, s = blockIdx.z;
    const Span span = batch_span(batch, s);
    const int64_t units = units_of(span);
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const Unit unit = unit_of(span, u);
        const uint32_t from = unit.from, count = unit.to - unit.from;
        const uint8_t* part = page_part<D, Q4>(cache, batch, s, unit.base, h);
        const uint32_t slot0 = part ? (uint32_t)(unit.base % cache.page_size) : 0;
        auto scale = [&](int which, uint32_t at) __attribute__((always_inline)) {
            return *reinterpret_cast<const uint32_t*>(part +
                Layout::scales(cache.page_size, which) + 4 * (slot0 + at));
        };
        auto value = [](uint32_t code, uint32_t word) __attribute__((always_inline)) {
            return __builtin_fmaf((float)code, bf16_to_f32(word & 0xffffu),
                bf16_to_f32(word >> 16));
        };
        // Keys: eight dims of a position at a time.
        for (uint32_t i = threadIdx.x; keys && i < count * (D / 8); i += 256) {
            const uint32_t t = i / (D / 8), c = i % (D / 8);
            float4 x, y;
            if (!part) {
                x.x = x.y = x.z = x.w = __builtin_nanf("");
                y = x;
            } else {
                const uint8_t* at = part + Layout::key_chunk(slot0 + from + t, c);
                float f[8];
                if (Q4) {
                    const uint32_t codes = *reinterpret_cast<const uint32_t*>(at);
                    const uint32_t word = scale(0, from + t);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        f[e] = value(codes >> nibble_at(e) & 15u, word);
                    }
                } else {
                    const f16x8 halves = *reinterpret_cast<const f16x8*>(at);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        f[e] = (float)halves[e];
                    }
                }
                x = make_float4(f[0], f[1], f[2], f[3]);
                y = make_float4(f[4], f[5], f[6], f[7]);
            }
            float* out = keys + (unit.token + t) * k_stride + (size_t)h * D + 8 * c;
            store4(out, x);
            store4(out + 4, y);
        }
        if (!values) {
            continue;
        }
        if (u != blockIdx.x) {
            __syncthreads();   // the previous unit's readers
        }
        // Values: a dim of eight positions at a time, through LDS.
        for (uint32_t i = threadIdx.x; part && i < 4 * D; i += 256) {
            const uint32_t d = i % D, g = i / D;
            bool any = false;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t at = 4 * g + (e & 3) + 16 * (e >> 2);
                any |= at >= from && at < from + count;
            }
            if (!any) {
                continue;
            }
            const uint8_t* at = part + Layout::values(cache.page_size) +
                Layout::value_chunk(slot0, d, g);
            if (Q4) {
                const uint32_t codes = *reinterpret_cast<const uint32_t*>(at);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    rows[4 * g + (e & 3) + 16 * (e >> 2)][d] = (float)(codes >> nibble_at(e) & 15u);
                }
            } else {
                const f16x8 halves = *reinterpret_cast<const f16x8*>(at);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    rows[4 * g + (e & 3) + 16 * (e >> 2)][d] = (float)halves[e];
                }
            }
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < count * D; i += 256) {
            const uint32_t t = i / D, d = i % D;
            float v = __builtin_nanf("");
            if (part) {
                v = rows[from + t][d];
                if (Q4) {
                    const uint32_t word = scale(1, from + t);
                    v = __builtin_fmaf(v, bf16_to_f32(word & 0xffffu), bf16_to_f32(word >> 16));
                }
            }
            values[(unit.token + t) * v_stride + (size_t)h * D + d] = v;
        }
    }
}

}  // namespace lh

using namespace lh;

// Units of the longest sequence's tokens.
static uint32_t unit_bound(const lh_paged_batch* b)
{
    const uint32_t query = b->max_query < b->tokens ? b->max_query : b->tokens;
    return query == 1 ? 1 : (query + 30) / 32 + 1;
}

template <int D, bool Q4>
static void append(const lh_paged_cache* c, const lh_paged_batch* b, const lh_append_rows* rows,
    hipStream_t s)
{
    const uint32_t units = unit_bound(b);
    hipLaunchKernelGGL((k_paged_append<D, Q4>),
        dim3(units, c->kv_heads * (rows->group ? 2 : 1), b->sequences), dim3(256), 0, s,
        pages_of(c), batch_of(b), *rows);
}

template <int D, bool Q4>
static void read(const lh_paged_cache* c, const lh_paged_batch* b, float* keys, size_t k_stride,
    float* values, size_t v_stride, hipStream_t s)
{
    const uint32_t units = unit_bound(b);
    hipLaunchKernelGGL((k_paged_read<D, Q4>), dim3(units, c->kv_heads, b->sequences), dim3(256), 0,
        s, pages_of(c), batch_of(b), keys, k_stride, values, v_stride);
}

extern "C" int lh_launch_paged_append(const lh_paged_cache* cache, const lh_paged_batch* batch,
    const lh_append_rows* rows, hipStream_t s)
{
    LH_FOR_CACHE(cache, append, cache, batch, rows, s);
    return (int)hipGetLastError();
}

extern "C" int lh_launch_paged_read(const lh_paged_cache* cache, const lh_paged_batch* batch,
    float* keys, size_t k_stride, float* values, size_t v_stride, hipStream_t s)
{
    LH_FOR_CACHE(cache, read, cache, batch, keys, k_stride, values, v_stride, s);
    return (int)hipGetLastError();
}
