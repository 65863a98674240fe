// Causal attention over the paged KV cache (lh_paged_attention), on the 16x16x32
// FP16 matrix instructions.
//
// The columns of the products are query rows: a sequence's (token, head of the KV
// head's group) pairs in turn, so a decode step fills them with a group's heads and
// a prompt with tokens of all of them. A wave takes blocks of 32 positions:
//   scores^T [32 positions][16 rows] = K Q^T, in two tiles of 16 positions;
//   out^T [D][16 rows] += V^T P^T.
// A lane holds four positions of either score tile for its column, which is exactly
// the operand that the second product takes from it (values lie in the pages in
// that order of positions), so the probabilities never leave the lane. One pass:
// running maximum and sum for each column, the four lanes of a column joined by two
// lane swaps for the maximum and once at the end for the sum.
//
// Precision: q (scaled by a power of two for each row) and p go in as two FP16 planes
// h + l, 22 bits or more; keys and values are exact FP16 numbers; sums are FP32.
// For 4-bit codes the products take code - 8, and
//   q.k = s (q.(c - 8)) + (z + 8 s) sum(q),  p v = (p s)(c - 8) + p (z + 8 s),
// so a scale is one multiplication for each position and never rounds a value.
#include "lh_paged.h"
#include "lh_mfma.h"

namespace lh {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f16x8 codes_minus8(uint32_t w)
{
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        // 0x6400 | c is 1024 + c.
        const f16x2 v = __builtin_bit_cast(f16x2, ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u);
        r[i] = __builtin_bit_cast(uint32_t, v - (f16x2){(_Float16)1032, (_Float16)1032});
    }
    return __builtin_bit_cast(f16x8, r);
}

// v as two FP16 planes: hi nearest to v, lo nearest to the rest. The rest has to be
// that of the hi which goes into the product: left to itself the compiler forms one
// by a fused multiplication and conversion and the other from the rounded product,
// and the two differ by a whole step at a tie (1 of 2^13 values). The empty asm
// makes the packed bits one value.
__device__ __forceinline__ void planes8(const float* v, f16x8& hi, f16x8& lo)
{
    u32x4 h, l;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t two = __builtin_bit_cast(uint32_t,
            (f16x2){(_Float16)v[2 * i], (_Float16)v[2 * i + 1]});
        asm("" : "+v"(two));
        h[i] = two;
        const f16x2 back = __builtin_bit_cast(f16x2, two);
        const f16x2 rest = {(_Float16)__builtin_fmaf((float)back[0], -1.0f, v[2 * i]),
            (_Float16)__builtin_fmaf((float)back[1], -1.0f, v[2 * i + 1])};
        l[i] = __builtin_bit_cast(uint32_t, rest);
    }
    hi = __builtin_bit_cast(f16x8, h);
    lo = __builtin_bit_cast(f16x8, l);
}

// Over the four lanes l % 16 of a column, in each of them.
__device__ __forceinline__ float column_max(float v)
{
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
        false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
        false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float column_sum(float v)
{
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
        false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
        false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

struct AttentionArgs {
    Pages cache;
    Batch batch;
    const float* q;
    float *out, *part;
    size_t q_stride, out_stride;
    uint64_t per_page;    // ceil(2^32 / (page_size / 32)): block -> page
    float scale;          // of the scores, times log2 e
    uint32_t group, splits;
    int vector_q;         // rows of q on 16-byte boundaries
};

// A 32-position block's loads: keys as [position tile][..], values, and (Q4) the
// words of the lane's positions 4 g .. + 3 and 16 + 4 g .. + 3.
template <int D, bool Q4>
struct KVBlock {
    static constexpr int N = Q4 ? D / 64 : D / 16;   // 16-byte words of keys, and of values
    u32x4 k[N], v[N], ks[2], vs[2];

    __device__ __forceinline__ void load(const uint8_t* part, uint32_t page_size, uint32_t slot,
        uint32_t lane)
    {
        typedef PageLayout<D, Q4> Layout;
        const uint32_t at = slot * Layout::vector;
        const u32x4* key = reinterpret_cast<const u32x4*>(part + at);
        const u32x4* value = reinterpret_cast<const u32x4*>(part + Layout::values(page_size) + at);
        if (Q4 && D == 64) {
            // Two 16-position tiles of 8 bytes a lane.
            const uint2 a = reinterpret_cast<const uint2*>(key)[lane];
            const uint2 b = reinterpret_cast<const uint2*>(key)[64 + lane];
            k[0] = (u32x4){a.x, a.y, b.x, b.y};
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) {
                k[i] = key[64 * i + lane];
            }
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i] = value[64 * i + lane];
        }
        if (Q4) {
            const uint32_t g = lane >> 4;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                ks[t] = *reinterpret_cast<const u32x4*>(part + Layout::scales(page_size, 0) +
                    4 * (slot + 16 * t + 4 * g));
                vs[t] = *reinterpret_cast<const u32x4*>(part + Layout::scales(page_size, 1) +
                    4 * (slot + 16 * t + 4 * g));
            }
        }
    }
    // Operand of position tile t's dims 32 j .. + 31.
    __device__ __forceinline__ f16x8 key(int t, int j) const
    {
        if (Q4) {
            const int w = t * (D / 32) + j;
            return codes_minus8(k[w >> 2][w & 3]);
        }
        return __builtin_bit_cast(f16x8, k[t * (D / 32) + j]);
    }
    __device__ __forceinline__ f16x8 value(int i) const
    {
        return Q4 ? codes_minus8(v[i >> 2][i & 3]) : __builtin_bit_cast(f16x8, v[i]);
    }
};

// Running state of a wave's NQ tiles of 16 columns.
template <int D, bool Q4, int NQ>
struct Columns {
    f16x8 hi[NQ][D / 32], lo[NQ][D / 32];   // q in planes
    float cs[NQ], qs[NQ];     // score factor, sum of the scaled q
    int32_t limit[NQ];        // last position that the column sees
    floatx4 acc[NQ][D / 16];  // out^T dims 16 i + 4 g .. + 3, times 2^14 (Q4: shift)
    float m[NQ], sum[NQ], offset[NQ];   // this lane's parts of the last two
    bool lost[NQ];
    int32_t low, high;        // least and largest limit of the wave
    float shift;              // Q4: 2^(13 - exponent of the largest value scale)

    __device__ __forceinline__ void block(const KVBlock<D, Q4>& b, int32_t base, uint32_t g)
    {
        const bool edge = base + 31 > low;
        float ks[8], kz[8], vs[8], vz[8];
        if (Q4) {
            float most = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t kw = b.ks[e >> 2][e & 3], vw = b.vs[e >> 2][e & 3];
                ks[e] = bf16_to_f32(kw & 0xffffu);
                kz[e] = __builtin_fmaf(8.0f, ks[e], __uint_as_float(kw & 0xffff0000u));
                vs[e] = bf16_to_f32(vw & 0xffffu);
                vz[e] = __builtin_fmaf(8.0f, vs[e], __uint_as_float(vw & 0xffff0000u));
                // Places past every column's limit may hold anything.
                const int32_t p = base + 4 * (int32_t)g + (e & 3) + 16 * (e >> 2);
                most = fmaxf(most, !edge || p <= high ? vs[e] : 0.0f);
            }
            // shift * vs stays below 2^14; a larger scale than so far lowers it.
            if (__ballot(most * shift >= 16384.0f)) {
                const float all = column_max(most);
                const int e = (int)((__float_as_uint(all) >> 23) & 0xffu) - 127;
                const float next = exp2i(e < -110 ? 123 : 13 - e);
                const float ratio = next / shift;
#pragma unroll
                for (int n = 0; n < NQ; n++) {
#pragma unroll
                    for (int i = 0; i < D / 16; i++) {
                        acc[n][i] *= ratio;
                    }
                }
                shift = next;
            }
        }
        floatx4 s[NQ][2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                s[n][t] = (floatx4){0, 0, 0, 0};
            }
#pragma unroll
            for (int j = 0; j < D / 32; j++) {
                const f16x8 k = b.key(t, j);
#pragma unroll
                for (int n = 0; n < NQ; n++) {
                    s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, hi[n][j], s[n][t], 0, 0, 0);
                    s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, lo[n][j], s[n][t], 0, 0, 0);
                }
            }
        }
        f16x8 ph[NQ], pl[NQ];
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            float p[8];
            uint32_t seen = 0xff;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float v = s[n][e >> 2][e & 3];
                v = Q4 ? __builtin_fmaf(kz[e], qs[n], ks[e] * v) : v;
                p[e] = v * cs[n];
            }
            if (edge) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const bool hidden = base + 4 * (int32_t)g + (e & 3) + 16 * (e >> 2) > limit[n];
                    p[e] = hidden ? -__builtin_inff() : p[e];
                    seen &= hidden ? ~(1u << e) : ~0u;
                }
            }
            float most = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])),
                fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
            most = fmaxf(column_max(most), m[n]);
            if (__ballot(most > m[n])) {
                const float keep = m[n] > -__builtin_inff() ? __builtin_amdgcn_exp2f(m[n] - most)
                    : 0.0f;
                m[n] = most;
                sum[n] *= keep;
                offset[n] *= keep;
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    acc[n][i] *= keep;
                }
            }
            const float top = m[n] > -__builtin_inff() ? m[n] : 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                p[e] = __builtin_amdgcn_exp2f(p[e] - top);
                sum[n] += p[e];
                if (Q4) {
                    const bool on = !edge || (seen >> e & 1);
                    offset[n] = __builtin_fmaf(p[e], on ? vz[e] : 0.0f, offset[n]);
                    p[e] *= on ? vs[e] * shift : 0.0f;
                } else {
                    p[e] *= 16384.0f;
                }
            }
            planes8(p, ph[n], pl[n]);
        }
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            f16x8 v = b.value(i);
            if (!Q4 && edge) {
                // An Inf or NaN at a position that some column does not see (or that
                // holds no value yet): out of the product, NaN for those that see it.
                f16x8 odd;
                bool any = false;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const bool bad = !__builtin_isfinite((float)v[e]);
                    const int32_t p = base + 4 * (int32_t)g + (e & 3) + 16 * (e >> 2);
                    odd[e] = bad && p <= high ? (_Float16)1 : (_Float16)0;
                    any |= bad && p <= high;
                    v[e] = bad ? (_Float16)0 : v[e];
                }
                if (__ballot(any)) {
#pragma unroll
                    for (int n = 0; n < NQ; n++) {
                        f16x8 on;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const int32_t p = base + 4 * (int32_t)g + (e & 3) + 16 * (e >> 2);
                            on[e] = p <= limit[n] ? (_Float16)1 : (_Float16)0;
                        }
                        const floatx4 none = {0, 0, 0, 0};
                        const floatx4 hits = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, on, none,
                            0, 0, 0);
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            acc[n][i][r] = hits[r] > 0 ? __builtin_nanf("") : acc[n][i][r];
                        }
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                acc[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[n], acc[n][i], 0, 0, 0);
                acc[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl[n], acc[n][i], 0, 0, 0);
            }
        }
    }
};

// Four waves take every fourth block of a split's range for one tile of 16 NQ
// query rows of a KV head. grid (KV heads, tiles * splits, sequences): the tiles of
// a KV head of eight share an XCD and its L2.
template <int D, bool Q4, int NQ>
__global__ void __launch_bounds__(256)
k_paged_attention(AttentionArgs a)
{
    constexpr int TQ = 16 * NQ, ROW = D + 4;
    __shared__ float joined[4][TQ][ROW];
    __shared__ float stats[4][3][TQ];
    const uint32_t h = blockIdx.x, s = blockIdx.z;
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, wave = threadIdx.x >> 6;
    const uint32_t split = blockIdx.y % a.splits;
    const Span span = batch_span(a.batch, s);
    const int64_t rows = span.count * a.group;
    const int64_t capacity = (int64_t)a.batch.width * a.cache.page_size;
    const uint32_t in_page = a.cache.page_size / 32;
    const int32_t* table = a.batch.table + (size_t)s * a.batch.width;
    const size_t head_bytes = PageLayout<D, Q4>::head_bytes(a.cache.page_size);
    for (int64_t tile = blockIdx.y / a.splits; tile * TQ < rows; tile += gridDim.y / a.splits) {
        Columns<D, Q4, NQ> c;
        c.low = 0x7fffffff;
        c.high = -1;
        c.shift = exp2i(123);
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            // Columns past the last row repeat it and are not stored.
            int64_t row = tile * TQ + 16 * n + (lane & 15);
            row = row < rows ? row : rows - 1;
            const int64_t t = row / a.group, last = span.first + t;
            c.lost[n] = last >= capacity;
            c.limit[n] = last < 0 ? -1 : (int32_t)(last < capacity ? last : capacity - 1);
            const float* q = a.q + (size_t)(span.begin + t) * a.q_stride +
                ((size_t)h * a.group + row % a.group) * D + 8 * g;
            float v[D / 4];
#pragma unroll
            for (int j = 0; j < D / 32; j++) {
                if (a.vector_q) {
                    const float4 x = *reinterpret_cast<const float4*>(q + 32 * j);
                    const float4 y = *reinterpret_cast<const float4*>(q + 32 * j + 4);
                    v[8 * j] = x.x, v[8 * j + 1] = x.y, v[8 * j + 2] = x.z, v[8 * j + 3] = x.w;
                    v[8 * j + 4] = y.x, v[8 * j + 5] = y.y, v[8 * j + 6] = y.z;
                    v[8 * j + 7] = y.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        v[8 * j + e] = q[32 * j + e];
                    }
                }
            }
            float most = 0, sum = 0;
#pragma unroll
            for (int e = 0; e < D / 4; e++) {
                most = fmaxf(most, fabsf(v[e]));
            }
            const int e2 = row_exponent(column_max(most));
            const float up = exp2i(e2);
#pragma unroll
            for (int e = 0; e < D / 4; e++) {
                v[e] *= up;
                sum += v[e];
            }
#pragma unroll
            for (int j = 0; j < D / 32; j++) {
                planes8(v + 8 * j, c.hi[n][j], c.lo[n][j]);
            }
            c.qs[n] = column_sum(sum);
            c.cs[n] = a.scale * exp2i(-e2);
            c.m[n] = -__builtin_inff();
            c.sum[n] = c.offset[n] = 0;
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                c.acc[n][i] = (floatx4){0, 0, 0, 0};
            }
        }
        // Limits do not fall from a column to the next.
        c.low = __builtin_amdgcn_readlane(c.limit[0], 0);
        c.high = __builtin_amdgcn_readlane(c.limit[NQ - 1], 15);
        const int32_t blocks = c.high < 0 ? 0 : (c.high >> 5) + 1;
        const int32_t chunk = (int32_t)(((int64_t)blocks + a.splits - 1) / a.splits);
        int32_t end = (int32_t)split * chunk + chunk;
        end = end < blocks ? end : blocks;
        for (int32_t b = (int32_t)split * chunk + (int32_t)wave; b < end; b += 4) {
            const uint32_t page = (uint32_t)((uint64_t)(uint32_t)b * a.per_page >> 32);
            const int32_t id = __builtin_amdgcn_readfirstlane(table[page]);
            if (id < 0 || (uint32_t)id >= a.cache.pages) {
#pragma unroll
                for (int n = 0; n < NQ; n++) {
                    c.lost[n] |= 32 * b <= c.limit[n];
                }
                continue;
            }
            const uint8_t* part = a.cache.base + ((size_t)id * a.cache.kv_heads + h) * head_bytes;
            KVBlock<D, Q4> kv;
            kv.load(part, a.cache.page_size, 32 * ((uint32_t)b - page * in_page), lane);
            c.block(kv, 32 * b, g);
        }
        // The four waves' parts: each scales its own to the common maximum.
        __syncthreads();   // the previous tile's readers
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            const float sum = column_sum(c.sum[n]), offset = column_sum(c.offset[n]);
            c.sum[n] = c.lost[n] ? __builtin_nanf("") : sum;
            c.offset[n] = offset;
            if (g == 0) {
                stats[wave][0][16 * n + lane] = c.m[n];
            }
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            const uint32_t col = 16 * n + (lane & 15);
            const float m = fmaxf(fmaxf(stats[0][0][col], stats[1][0][col]),
                fmaxf(stats[2][0][col], stats[3][0][col]));
            const float keep = c.m[n] > -__builtin_inff() ? __builtin_amdgcn_exp2f(c.m[n] - m)
                : 0.0f;
            // 1 / shift is a power of two.
            const float back = keep * (Q4 ? 1.0f / c.shift : 1.0f / 16384);
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                floatx4 v;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    v[r] = __builtin_fmaf(c.acc[n][i][r], back, Q4 ? c.offset[n] * keep : 0.0f);
                }
                *reinterpret_cast<floatx4*>(&joined[wave][col][16 * i + 4 * g]) = v;
            }
            if (g == 0) {
                stats[wave][1][col] = c.lost[n] ? __builtin_nanf("") : c.sum[n] * keep;
                stats[wave][2][col] = m;
            }
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < TQ * D; i += 256) {
            const uint32_t col = i / D, d = i % D;
            const int64_t row = tile * TQ + col;
            if (row >= rows) {
                break;
            }
            const float v = (joined[0][col][d] + joined[1][col][d]) +
                (joined[2][col][d] + joined[3][col][d]);
            const float sum = (stats[0][1][col] + stats[1][1][col]) +
                (stats[2][1][col] + stats[3][1][col]);
            const size_t token = (size_t)(span.begin + row / a.group);
            const size_t head = (size_t)h * a.group + row % a.group;
            if (a.splits == 1) {
                // No position at all: 0.
                a.out[token * a.out_stride + head * D + d] = sum == 0 ? 0.0f : v / sum;
            } else {
                const size_t at = (token * a.cache.kv_heads * a.group + head) * a.splits + split;
                float* part = a.part + at * (D + 2);
                part[2 + d] = v;
                if (d == 0) {
                    part[0] = stats[0][2][col];
                    part[1] = sum;
                }
            }
        }
    }
}

// Joins the splits of a (token, head): one workgroup of D threads each.
template <int D>
__global__ void __launch_bounds__(D)
k_paged_join(AttentionArgs a)
{
    const uint32_t head = blockIdx.x, s = blockIdx.z, d = threadIdx.x;
    const uint32_t heads = a.cache.kv_heads * a.group;
    const Span span = batch_span(a.batch, s);
    for (int64_t t = blockIdx.y; t < span.count; t += gridDim.y) {
        const size_t token = (size_t)(span.begin + t);
        const float* part = a.part + (token * heads + head) * a.splits * (D + 2);
        float m = -__builtin_inff();
        for (uint32_t i = 0; i < a.splits; i++) {
            m = fmaxf(m, part[(size_t)i * (D + 2)]);
        }
        float sum = 0, v = 0;
#pragma unroll 4
        for (uint32_t i = 0; i < a.splits; i++) {
            const float* p = part + (size_t)i * (D + 2);
            // A split that saw nothing holds sums of 0, or NaN for a lost position.
            const float keep = p[0] > -__builtin_inff() ? __builtin_amdgcn_exp2f(p[0] - m) : 1.0f;
            sum = __builtin_fmaf(p[1], keep, sum);
            v = __builtin_fmaf(p[2 + d], keep, v);
        }
        a.out[token * a.out_stride + (size_t)head * D + d] = sum == 0 ? 0.0f : v / sum;
    }
}

}  // namespace lh

using namespace lh;

// Workgroups that fill the chip: two of four waves on each of its 256 units.
enum { ATTENTION_WORKGROUPS = 512 };

struct AttentionPlan {
    uint32_t tiles, splits, wide;   // wide: two tiles of 16 rows a wave
};

static AttentionPlan attention_plan(const lh_paged_cache* c, const lh_paged_batch* b,
    uint32_t group)
{
    const uint64_t query = b->max_query < b->tokens ? b->max_query : b->tokens;
    const uint64_t rows = query * group;
    AttentionPlan p;
    p.wide = rows > 16;
    const uint64_t tile = p.wide ? 32 : 16, tiles = (rows + tile - 1) / tile;
    p.tiles = (uint32_t)(tiles < 1024 ? tiles : 1024);
    uint64_t longest = (uint64_t)b->table_width * c->page_size;
    longest = b->max_length < longest ? b->max_length : longest;
    const uint64_t blocks = (longest + 31) / 32;
    const uint64_t groups = (uint64_t)p.tiles * c->kv_heads * b->sequences;
    // Two blocks a wave at least: less does not pay the join.
    uint64_t splits = ATTENTION_WORKGROUPS / groups, most = (blocks + 7) / 8;
    splits = splits < most ? splits : most;
    p.splits = (uint32_t)(splits < 1 ? 1 : splits > 63 ? 63 : splits);
    return p;
}

extern "C" size_t lh_paged_attention_scratch_bytes(const lh_paged_cache* cache,
    const lh_paged_batch* batch, uint32_t group)
{
    const AttentionPlan p = attention_plan(cache, batch, group);
    if (p.splits == 1) {
        return 0;
    }
    return lh_round16((size_t)batch->tokens * cache->kv_heads * group * p.splits *
        (cache->head_dim + 2) * 4);
}

template <int D, bool Q4>
static void attention(const lh_paged_cache* c, const lh_paged_batch* b, const AttentionPlan& p,
    const AttentionArgs& a, hipStream_t s)
{
    const dim3 grid(c->kv_heads, p.tiles * p.splits, b->sequences);
    if (p.wide) {
        hipLaunchKernelGGL((k_paged_attention<D, Q4, 2>), grid, dim3(256), 0, s, a);
    } else {
        hipLaunchKernelGGL((k_paged_attention<D, Q4, 1>), grid, dim3(256), 0, s, a);
    }
    if (p.splits > 1) {
        const uint32_t query = b->max_query < b->tokens ? b->max_query : b->tokens;
        hipLaunchKernelGGL((k_paged_join<D>), dim3(c->kv_heads * a.group,
            query < 65535 ? query : 65535, b->sequences), dim3(D), 0, s, a);
    }
}

extern "C" int lh_launch_paged_attention(const lh_paged_cache* cache, const lh_paged_batch* batch,
    uint32_t group, const float* q, size_t q_stride, float scale, float* out, size_t out_stride,
    uint8_t* scratch, hipStream_t s)
{
    const AttentionPlan p = attention_plan(cache, batch, group);
    const uint32_t in_page = cache->page_size / 32;
    const AttentionArgs a = {pages_of(cache), batch_of(batch), q, out,
        reinterpret_cast<float*>(scratch), q_stride, out_stride,
        (((uint64_t)1 << 32) + in_page - 1) / in_page, scale * 1.44269504088896341f, group,
        p.splits, ((uintptr_t)q & 15) == 0 && q_stride % 4 == 0};
    LH_FOR_CACHE(cache, attention, cache, batch, p, a, s);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
