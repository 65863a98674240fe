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
#include "lh_nibbles.h"
#include "lh_paged.h"

namespace lh {

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
    float *out, *part;    // part [row][split][D]: a split's sums of values
    float2* tops;         // [row][split]: its maximum and sum of probabilities
    size_t q_stride, out_stride;
    uint64_t per_page;    // ceil(2^32 / (page_size / 32)): block -> page
    float scale;          // of the scores, times log2 e
    uint32_t group, splits, tiles;
    uint32_t chunk, tile;   // 64-position steps of a split, rows of a tile
};

// Steps of each split of a row tile that sees `steps`: the planned number, or more
// where a sequence is longer than the plan's bound.
__device__ __forceinline__ int32_t split_chunk(const AttentionArgs& a, int32_t steps)
{
    const int32_t even = (int32_t)(((int64_t)steps + a.splits - 1) / a.splits);
    return even > (int32_t)a.chunk ? even : (int32_t)a.chunk;
}

// A lane's part of a query row: dims 32 j + 8 g .. + 7, scaled by a power of two so
// that the row's largest lies in [2^14, 2^15), in planes; cs takes a score in units
// of that back (times log2 e), qs is the row's sum in them.
template <int D>
__device__ __forceinline__ void load_query(const float* q, uint32_t g, float scale,
    f16x8 (&hi)[D / 32], f16x8 (&lo)[D / 32], float& cs, float& qs)
{
    float v[D / 4];
    q += 8 * g;
#pragma unroll
    for (int j = 0; j < D / 32; j++) {
        const float4 x = load4(q + 32 * j), y = load4(q + 32 * j + 4);
        v[8 * j] = x.x, v[8 * j + 1] = x.y, v[8 * j + 2] = x.z, v[8 * j + 3] = x.w;
        v[8 * j + 4] = y.x, v[8 * j + 5] = y.y, v[8 * j + 6] = y.z, v[8 * j + 7] = y.w;
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
        planes8(v + 8 * j, hi[j], lo[j]);
    }
    qs = column_sum(sum);
    cs = scale * exp2i(-e2);
}

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
    __device__ __forceinline__ f16x8 key(int t, int j, const NibbleMasks& mask) const
    {
        if (Q4) {
            const int w = t * (D / 32) + j;
            return codes_minus8(k[w >> 2][w & 3], mask);
        }
        return __builtin_bit_cast(f16x8, k[t * (D / 32) + j]);
    }
    __device__ __forceinline__ f16x8 value(int i, const NibbleMasks& mask) const
    {
        return Q4 ? codes_minus8(v[i >> 2][i & 3], mask) : __builtin_bit_cast(f16x8, v[i]);
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
    NibbleMasks mask;

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
                const f16x8 k = b.key(t, j, mask);
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
            f16x8 v = b.value(i, mask);
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
// query rows of a KV head. grid (KV heads, sequences, tiles of the splits in turn): the
// tiles of a KV head of eight share an XCD and its L2.
template <int D, bool Q4, int NQ>
__global__ void __launch_bounds__(256)
k_paged_attention(AttentionArgs a)
{
    constexpr int TQ = 16 * NQ, ROW = D + 4;
    __shared__ float joined[4][TQ][ROW];
    __shared__ float stats[4][3][TQ];
    const uint32_t h = blockIdx.x, s = blockIdx.y;
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t split = blockIdx.z / a.tiles;
    const Span span = batch_span(a.batch, s);
    const int64_t rows = span.count * a.group;
    const int64_t capacity = (int64_t)a.batch.width * a.cache.page_size;
    const uint32_t in_page = a.cache.page_size / 32;
    const int32_t* table = a.batch.table + (size_t)s * a.batch.width;
    const size_t head_bytes = PageLayout<D, Q4>::head_bytes(a.cache.page_size);
    for (int64_t tile = blockIdx.z % a.tiles; tile * TQ < rows; tile += a.tiles) {
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
                ((size_t)h * a.group + row % a.group) * D;
            load_query<D>(q, g, a.scale, c.hi[n], c.lo[n], c.cs[n], c.qs[n]);
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
        const int32_t steps = c.high < 0 ? 0 : (c.high >> 6) + 1;
        const int32_t blocks = c.high < 0 ? 0 : (c.high >> 5) + 1;
        const int32_t chunk = split_chunk(a, steps);
        if (split && (int64_t)split * chunk >= steps) {
            continue;   // nothing for this split: the join does not ask for it
        }
        const int32_t first = 2 * (int32_t)split * chunk;
        const int32_t end = blocks - first < 2 * chunk ? blocks : first + 2 * chunk;
        for (int32_t b = first + (int32_t)wave; b < end; b += 4) {
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
            if (steps <= chunk) {
                // No position at all: 0.
                a.out[token * a.out_stride + head * D + d] = sum == 0 ? 0.0f : v / sum;
            } else {
                const size_t at = (token * a.cache.kv_heads * a.group + head) * a.splits + split;
                a.part[at * D + d] = v;
                if (d == 0) {
                    a.tops[at] = make_float2(stats[0][2][col], sum);
                }
            }
        }
    }
}

// What a lane holds of a step of 64 positions (two blocks): keys and values as they lie
// in the pages and (Q4) the scale words of its own positions, 4 g .. + 3 of every
// PACK-th 16-position tile.
template <int D, bool Q4, int C>
struct DecodeStep {
    static constexpr int PACK = 16 / C;
    static constexpr int N = Q4 ? D / 64 : D / 16;   // 16-byte words of a block's keys
    u32x4 k[2][N], v[2][N], ks[C / 4], vs[C / 4];

    // part: the KV head's part of the two blocks' pages, slot: the blocks' places there.
    __device__ __forceinline__ void load_keys(const uint8_t* const (&part)[2],
        const uint32_t (&slot)[2], uint32_t page_size, uint32_t lane)
    {
        typedef PageLayout<D, Q4> Layout;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const u32x4* key = reinterpret_cast<const u32x4*>(part[b] + slot[b] * Layout::vector);
            if (Q4 && D == 64) {
                // Two tiles of 8 bytes a lane.
                const uint2 x = reinterpret_cast<const uint2*>(key)[lane];
                const uint2 y = reinterpret_cast<const uint2*>(key)[64 + lane];
                k[b][0] = (u32x4){x.x, x.y, y.x, y.y};
            } else {
#pragma unroll
                for (int i = 0; i < N; i++) {
                    k[b][i] = key[64 * i + lane];
                }
            }
        }
        if (Q4) {
            load_words(ks, 0, part, slot, page_size, lane);
        }
    }
    __device__ __forceinline__ void load_values(const uint8_t* const (&part)[2],
        const uint32_t (&slot)[2], uint32_t page_size, uint32_t lane)
    {
        typedef PageLayout<D, Q4> Layout;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const u32x4* value = reinterpret_cast<const u32x4*>(part[b] +
                Layout::values(page_size) + slot[b] * Layout::vector);
#pragma unroll
            for (int i = 0; i < N; i++) {
                v[b][i] = value[64 * i + lane];
            }
        }
        if (Q4) {
            load_words(vs, 1, part, slot, page_size, lane);
        }
    }
    __device__ __forceinline__ void load_words(u32x4 (&to)[C / 4], int which,
        const uint8_t* const (&part)[2], const uint32_t (&slot)[2], uint32_t page_size,
        uint32_t lane)
    {
        typedef PageLayout<D, Q4> Layout;
        const uint32_t g = lane >> 4, u = (lane & 15) / C;
#pragma unroll
        for (int w = 0; w < C / 4; w++) {
            const uint32_t tile = PACK * w + u;
            const size_t second = tile >= 2 ? ~(size_t)0 : 0;
            const uint8_t* p = part[0] + (second & (size_t)(part[1] - part[0]));
            const uint32_t at = slot[0] + ((uint32_t)second & (slot[1] - slot[0])) +
                16 * (tile & 1) + 4 * g;
            to[w] = *reinterpret_cast<const u32x4*>(p + Layout::scales(page_size, which) + 4 * at);
        }
    }
};

// Decode: a wave takes steps of 64 positions (four tiles of 16) for at most C query
// rows (C = 4, 8 or 16), and every column of the products works: column r holds row
// r % C and keeps only the tiles with tile % (16 / C) = r / C, a softmax of its own over
// a part of the positions. So a lane forms C probabilities a step whatever C is,
// instead of 16; columns of one row meet where the waves and the splits do.
template <int D, bool Q4, int C>
struct Decode {
    static constexpr int PACK = 16 / C;              // columns of a row
    typedef DecodeStep<D, Q4, C> Step;
    // 128 dims of FP16 keys and values fill half of the registers: the planes of q then
    // stay in LDS, one copy for the four waves.
    static constexpr bool SHARED = !Q4 && D == 128;
    f16x8 hi[SHARED ? 1 : D / 32], lo[SHARED ? 1 : D / 32];
    const f16x8* planes;   // [hi, lo][j][lane]
    uint32_t lane;
    float cs, qs;
    int32_t limit, low, high;
    floatx4 acc[D / 16];
    float m, sum, offset, shift;
    bool lost;
    NibbleMasks mask;
    uint32_t g, u;   // lane / 16, lane % 16 / C

    __device__ __forceinline__ int32_t position(int32_t base, int e) const
    {
        return base + 16 * (PACK * (e >> 2) + (int32_t)u) + 4 * (int32_t)g + (e & 3);
    }

    // Scores of the lane's positions, in units of 2: s * scale * log2 e.
    __device__ __forceinline__ void scores(const Step& step, float (&p)[C])
    {
        floatx4 s[4];
        uint32_t at = lane;
        if (SHARED) {
            asm volatile("" : "+v"(at));   // read again each step, not kept
        }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            s[t] = (floatx4){0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < D / 32; j++) {
                const int w = (t & 1) * (D / 32) + j;
                const f16x8 x = Q4 ? codes_minus8(step.k[t >> 1][w >> 2][w & 3], mask)
                    : __builtin_bit_cast(f16x8, step.k[t >> 1][Q4 ? 0 : w]);
                const f16x8 qh = SHARED ? planes[64 * j + at] : hi[SHARED ? 0 : j];
                const f16x8 ql = SHARED ? planes[64 * (D / 32 + j) + at] : lo[SHARED ? 0 : j];
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, qh, s[t], 0, 0, 0);
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ql, s[t], 0, 0, 0);
            }
        }
#pragma unroll
        for (int w = 0; w < C / 4; w++) {
            floatx4 mine = s[PACK * w];
#pragma unroll
            for (int x = 1; x < PACK; x++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    mine[i] = u == (uint32_t)x ? s[PACK * w + x][i] : mine[i];
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float y = mine[i];
                if (Q4) {
                    const uint32_t word = step.ks[w][i];
                    const float scale = bf16_to_f32(word & 0xffffu);
                    const float z = __builtin_fmaf(8.0f, scale,
                        __uint_as_float(word & 0xffff0000u));
                    y = __builtin_fmaf(z, qs, scale * y);
                }
                p[4 * w + i] = y * cs;
            }
        }
    }

    // The softmax over the step and the operands of the second product: p (times the
    // value scales) in planes, pairs 0 and 1 of tile PACK * w + u in words 2 w and 2 w + 1.
    __device__ __forceinline__ void probabilities(const Step& step, float (&p)[C], int32_t base, bool edge,
        uint32_t (&ph)[C / 2], uint32_t (&pl)[C / 2])
    {
        float scale[C], z[C];
        if (Q4) {
            float most = 0;
#pragma unroll
            for (int e = 0; e < C; e++) {
                const uint32_t word = step.vs[e >> 2][e & 3];
                scale[e] = bf16_to_f32(word & 0xffffu);
                z[e] = __builtin_fmaf(8.0f, scale[e], __uint_as_float(word & 0xffff0000u));
                if (edge && position(base, e) > limit) {
                    scale[e] = z[e] = 0;   // may hold anything
                }
                most = fmaxf(most, scale[e]);
            }
            // shift * scale stays below 2^14; a larger scale than so far lowers it.
            if (__ballot(most * shift >= 16384.0f)) {
                most = column_max(most);
                const int e = (int)((__float_as_uint(most) >> 23) & 0xffu) - 127;
                const float next = fminf(shift, exp2i(e < -110 ? 123 : 13 - e));
                const float ratio = next / shift;
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    acc[i] *= ratio;
                }
                shift = next;
            }
        }
        if (edge) {
#pragma unroll
            for (int e = 0; e < C; e++) {
                p[e] = position(base, e) > limit ? -__builtin_inff() : p[e];
            }
        }
        float most = p[0];
#pragma unroll
        for (int e = 1; e < C; e++) {
            most = fmaxf(most, p[e]);
        }
        most = fmaxf(column_max(most), m);
        if (__ballot(most > m)) {
            const float keep = m > -__builtin_inff() ? __builtin_amdgcn_exp2f(m - most) : 0.0f;
            m = most;
            sum *= keep;
            offset *= keep;
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                acc[i] *= keep;
            }
        }
        const float top = m > -__builtin_inff() ? m : 0.0f;
#pragma unroll
        for (int e = 0; e < C; e++) {
            p[e] = __builtin_amdgcn_exp2f(p[e] - top);
            sum += p[e];
            if (Q4) {
                offset = __builtin_fmaf(p[e], z[e], offset);
                p[e] *= scale[e] * shift;
            } else {
                p[e] *= 16384.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < C / 2; i++) {
            planes2(p[2 * i], p[2 * i + 1], ph[i], pl[i]);
        }
    }

    // Block b's operand from the pairs: each half from the column that has its tile.
    __device__ __forceinline__ f16x8 operand(const uint32_t (&pair)[C / 2], int b) const
    {
        u32x4 x;
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const int tile = 2 * b + half, w = tile / PACK;
            const bool mine = PACK == 1 || u == (uint32_t)(tile % PACK);
            x[2 * half] = mine ? pair[2 * w] : 0;
            x[2 * half + 1] = mine ? pair[2 * w + 1] : 0;
        }
        return __builtin_bit_cast(f16x8, x);
    }

    __device__ __forceinline__ void products(const Step& step, const uint32_t (&ph)[C / 2],
        const uint32_t (&pl)[C / 2], int32_t base, bool edge)
    {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const f16x8 h = operand(ph, b), l = operand(pl, b);
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                f16x8 x = Q4 ? codes_minus8(step.v[b][i >> 2][i & 3], mask)
                    : __builtin_bit_cast(f16x8, step.v[b][Q4 ? 0 : i]);
                if (!Q4 && edge) {
                    x = without_odd(x, i, b, base);
                }
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, h, acc[i], 0, 0, 0);
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, l, acc[i], 0, 0, 0);
            }
        }
    }

    // x with every Inf or NaN as 0: it may stand at a position that some column does not
    // see, or that holds no value yet. Columns that see it get NaN.
    __device__ __forceinline__ f16x8 without_odd(f16x8 x, int i, int b, int32_t base)
    {
        f16x8 odd, on;
        bool any = false;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int32_t p = base + 32 * b + 4 * (int32_t)g + (e & 3) + 16 * (e >> 2);
            const bool bad = !__builtin_isfinite((float)x[e]);
            odd[e] = bad && p <= high ? (_Float16)1 : (_Float16)0;
            any |= bad && p <= high;
            x[e] = bad ? (_Float16)0 : x[e];
            on[e] = p <= limit ? (_Float16)1 : (_Float16)0;
        }
        if (__ballot(any)) {
            const floatx4 hits = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, on,
                (floatx4){0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                acc[i][r] = hits[r] > 0 ? __builtin_nanf("") : acc[i][r];
            }
        }
        return x;
    }
};

// Four waves take every fourth step of a split's range for C query rows of a KV
// head. grid (KV heads, sequences, tiles of the splits in turn): a KV head of eight has
// an XCD to itself, and splits come last because only long sequences have the later
// ones (with the splits of a sequence side by side, the full ones of four all fell on
// the same quarter of an XCD: 151 against 106 us for 64 sequences).
template <int D, bool Q4, int C>
__global__ void __launch_bounds__(256, C == 16 && D == 128 ? 1 : 2)
k_paged_decode(AttentionArgs a)
{
    constexpr int ROW = D + 4, PACK = 16 / C;
    __shared__ float joined[4][16][ROW];
    __shared__ float stats[4][2][16], tops[16];
    __shared__ f16x8 planes[Decode<D, Q4, C>::SHARED ? 2 * (D / 32) * 64 : 1];
    const uint32_t h = blockIdx.x, s = blockIdx.y, lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t split = blockIdx.z / a.tiles;
    const Span span = batch_span(a.batch, s);
    const int64_t rows = span.count * a.group;
    const int64_t capacity = (int64_t)a.batch.width * a.cache.page_size;
    const uint32_t in_page = a.cache.page_size / 32;
    const int32_t* table = a.batch.table + (size_t)s * a.batch.width;
    const size_t head_bytes = PageLayout<D, Q4>::head_bytes(a.cache.page_size);
    for (int64_t tile = blockIdx.z % a.tiles; tile * C < rows; tile += a.tiles) {
        Decode<D, Q4, C> c;
        c.planes = planes;
        c.lane = lane;
        c.g = lane >> 4;
        c.u = (lane & 15) / C;
        // Rows past the last one repeat it and are not stored.
        int64_t row = tile * C + (lane & 15) % C;
        row = row < rows ? row : rows - 1;
        const int64_t t = row / a.group, last = span.first + t;
        c.lost = last >= capacity;
        c.limit = last < 0 ? -1 : (int32_t)(last < capacity ? last : capacity - 1);
        // Limits do not fall from a row to the next.
        c.low = __builtin_amdgcn_readlane(c.limit, 0);
        c.high = __builtin_amdgcn_readlane(c.limit, C - 1);
        const int32_t steps = c.high < 0 ? 0 : (c.high >> 6) + 1;
        const int32_t chunk = split_chunk(a, steps);
        if (split && (int64_t)split * chunk >= steps) {
            continue;   // nothing for this split: the join does not ask for it
        }
        const int32_t first = (int32_t)split * chunk;
        const int32_t end = steps - first < chunk ? steps : first + chunk;
        c.m = -__builtin_inff();
        c.sum = c.offset = 0;
        c.shift = exp2i(123);
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            c.acc[i] = (floatx4){0, 0, 0, 0};
        }
        // Lane i has the page ids of the wave's steps 64 n + i.
        int32_t ids[2] = {0, 0};
        const uint8_t* part[2];
        uint32_t slot[2];
        // Places of step x; a block without a place reads page 0 and is lost for the
        // columns that see it.
        auto locate = [&](int32_t x, int32_t turn) __attribute__((always_inline)) {
            if ((turn & 63) == 0) {
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const int64_t block = 2 * ((int64_t)x + 4 * (int64_t)lane) + b;
                    const int64_t at = (int64_t)((uint64_t)block * a.per_page >> 32);
                    ids[b] = at < a.batch.width ? table[at] : -1;
                }
            }
#pragma unroll
            for (int b = 0; b < 2; b++) {
                const uint32_t block = 2 * (uint32_t)x + b;
                const uint32_t page = (uint32_t)((uint64_t)block * a.per_page >> 32);
                int32_t id = __builtin_amdgcn_readlane(ids[b], turn & 63);
                if (id < 0 || (uint32_t)id >= a.cache.pages) {
                    id = 0;
                    c.lost |= 32 * (int32_t)block <= c.limit;
                }
                slot[b] = 32 * (block - page * in_page);
                part[b] = a.cache.base + ((size_t)id * a.cache.kv_heads + h) * head_bytes;
            }
        };
        int32_t x = first + (int32_t)wave;
        DecodeStep<D, Q4, C> step;
        auto keys = [&](auto& to) __attribute__((always_inline)) { to.load_keys(part, slot, a.cache.page_size, lane); };
        auto values = [&](auto& to) __attribute__((always_inline)) { to.load_values(part, slot, a.cache.page_size, lane); };
        if (x < end) {
            locate(x, 0);
            keys(step);
            values(step);
        }
        const float* q = a.q + (size_t)(span.begin + t) * a.q_stride +
            ((size_t)h * a.group + row % a.group) * D;
        if constexpr (Decode<D, Q4, C>::SHARED) {
            f16x8 hi[D / 32], lo[D / 32];
            load_query<D>(q, c.g, a.scale, hi, lo, c.cs, c.qs);
            __syncthreads();   // the previous tile's readers
            if (wave == 0) {
#pragma unroll
                for (int j = 0; j < D / 32; j++) {
                    planes[64 * j + lane] = hi[j];
                    planes[64 * (D / 32 + j) + lane] = lo[j];
                }
            }
            __syncthreads();
        } else {
            load_query<D>(q, c.g, a.scale, c.hi, c.lo, c.cs, c.qs);
        }
        int32_t turn = 0;
        if constexpr (Q4) {
            // A step is little: the next one's loads run during all of this one.
            while (x < end) {
                const int32_t base = 64 * x;
                const bool edge = base + 63 > c.low;
                float p[C];
                uint32_t ph[C / 2], pl[C / 2];
                DecodeStep<D, Q4, C> next = step;
                x += 4;
                if (x < end) {
                    locate(x, ++turn);
                    keys(next);
                    values(next);
                }
                c.scores(step, p);
                c.probabilities(step, p, base, edge, ph, pl);
                c.products(step, ph, pl, base, edge);
                step = next;
            }
        } else {
            // Registers for one step: the next one's keys and values are asked for as soon
            // as this one's are done with.
            while (x < end) {
                const int32_t base = 64 * x;
                const bool edge = base + 63 > c.low;
                float p[C];
                uint32_t ph[C / 2], pl[C / 2];
                x += 4;
                c.scores(step, p);
                if (x < end) {
                    locate(x, ++turn);
                    keys(step);
                }
                c.probabilities(step, p, base, edge, ph, pl);
                c.products(step, ph, pl, base, edge);
                if (x < end) {
                    values(step);
                }
            }
        }
        // The waves' columns: each scales its own to its row's maximum.
        __syncthreads();   // the previous tile's readers
        c.sum = column_sum(c.sum);
        c.offset = column_sum(c.offset);
        if (c.g == 0) {
            stats[wave][0][lane] = c.m;
        }
        __syncthreads();
        float m = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < 4; w++) {
#pragma unroll
            for (int y = 0; y < PACK; y++) {
                m = fmaxf(m, stats[w][0][(lane & 15) % C + C * y]);
            }
        }
        const float keep = c.m > -__builtin_inff() ? __builtin_amdgcn_exp2f(c.m - m) : 0.0f;
        const float back = keep * (Q4 ? 1.0f / c.shift : 1.0f / 16384);   // powers of two
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            floatx4 y;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                y[r] = __builtin_fmaf(c.acc[i][r], back, Q4 ? c.offset * keep : 0.0f);
            }
            *reinterpret_cast<floatx4*>(&joined[wave][lane & 15][16 * i + 4 * c.g]) = y;
        }
        if (c.g == 0) {
            stats[wave][1][lane] = c.lost ? __builtin_nanf("") : c.sum * keep;
        }
        if (wave == 0 && lane < C) {
            tops[lane] = m;
        }
        __syncthreads();
        const bool whole = steps <= chunk;   // no other split has a part
        for (uint32_t i = threadIdx.x; i < C * D; i += 256) {
            const uint32_t col = i / D, d = i % D;
            const int64_t mine = tile * C + col;
            if (mine >= rows) {
                break;
            }
            float v = 0, sum = 0;
#pragma unroll
            for (int w = 0; w < 4; w++) {
#pragma unroll
                for (int y = 0; y < PACK; y++) {
                    v += joined[w][col + C * y][d];
                    sum += stats[w][1][col + C * y];
                }
            }
            const size_t token = (size_t)(span.begin + mine / a.group);
            const size_t head = (size_t)h * a.group + mine % a.group;
            if (whole) {
                // No position at all: 0.
                a.out[token * a.out_stride + head * D + d] = sum == 0 ? 0.0f : v / sum;
            } else {
                const size_t at = (token * a.cache.kv_heads * a.group + head) * a.splits + split;
                a.part[at * D + d] = v;
                if (d == 0) {
                    a.tops[at] = make_float2(tops[col], sum);
                }
            }
        }
    }
}

// Joins the splits of a (token, head): lane i of every wave weighs splits i, i + 64 ..
// (at most SPLITS), then 256 / (D / 4) groups of threads take every so many of them,
// four dims a thread.
enum { SPLITS = 256 };

template <int D>
__global__ void __launch_bounds__(256)
k_paged_join(AttentionArgs a)
{
    constexpr uint32_t QUADS = D / 4, GROUPS = 256 / QUADS;
    __shared__ float weight[SPLITS];
    __shared__ float4 joined[GROUPS][QUADS];
    const uint32_t head = blockIdx.x, s = blockIdx.z, lane = threadIdx.x & 63;
    const uint32_t heads = a.cache.kv_heads * a.group;
    const uint32_t quad = threadIdx.x % QUADS, group = threadIdx.x / QUADS;
    const Span span = batch_span(a.batch, s);
    const int64_t rows = span.count * a.group;
    const int64_t capacity = (int64_t)a.batch.width * a.cache.page_size;
    for (int64_t t = blockIdx.y; t < span.count; t += gridDim.y) {
        // The splits that the row's tile had.
        int64_t end = (t * a.group + head % a.group) / a.tile * a.tile + a.tile;
        end = end < rows ? end : rows;
        int64_t last = span.first + (end - 1) / a.group;
        last = last < capacity ? last : capacity - 1;
        const int32_t steps = last < 0 ? 0 : (int32_t)(last >> 6) + 1;
        const int32_t chunk = split_chunk(a, steps);
        if (steps <= chunk) {
            continue;   // written already
        }
        const uint32_t splits = (uint32_t)((steps + chunk - 1) / chunk);
        const size_t token = (size_t)(span.begin + t), row = (token * heads + head) * a.splits;
        float2 tops[SPLITS / 64];
        float m = -__builtin_inff(), sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < SPLITS / 64; i++) {
            tops[i] = lane + 64 * i < splits ? a.tops[row + lane + 64 * i]
                : make_float2(-__builtin_inff(), 0.0f);
            m = fmaxf(m, tops[i].x);
        }
        m = wave_max64(m);
#pragma unroll
        for (uint32_t i = 0; i < SPLITS / 64; i++) {
            // A split that saw nothing holds sums of 0, or NaN for a lost position.
            const float keep = tops[i].x > -__builtin_inff()
                ? __builtin_amdgcn_exp2f(tops[i].x - m) : 1.0f;
            sum = __builtin_fmaf(tops[i].y, keep, sum);
            if (threadIdx.x < 64) {
                weight[lane + 64 * i] = keep;
            }
        }
        sum = wave_lane0(wave_tree64(sum));
        __syncthreads();
        float4 v = make_float4(0, 0, 0, 0);
        const float4* part = reinterpret_cast<const float4*>(a.part) + row * QUADS + quad;
#pragma unroll 4
        for (uint32_t i = group; i < splits; i += GROUPS) {
            const float4 x = part[(size_t)i * QUADS];
            const float w = weight[i];
            v.x = __builtin_fmaf(x.x, w, v.x);
            v.y = __builtin_fmaf(x.y, w, v.y);
            v.z = __builtin_fmaf(x.z, w, v.z);
            v.w = __builtin_fmaf(x.w, w, v.w);
        }
        joined[group][quad] = v;
        __syncthreads();
        if (threadIdx.x < D) {
            const float* each = reinterpret_cast<const float*>(joined);
            float y = 0;
#pragma unroll
            for (uint32_t i = 0; i < GROUPS; i++) {
                y += each[i * D + threadIdx.x];
            }
            a.out[token * a.out_stride + (size_t)head * D + threadIdx.x] =
                sum == 0 ? 0.0f : y / sum;
        }
        __syncthreads();   // before the next row's weights
    }
}

}  // namespace lh

using namespace lh;

// How the steps are split. RESIDENT workgroups are on the chip at once; up to them a
// split takes as few as MIN_CHUNK steps (one sequence of 16000 positions: 13.7 us with
// 8, 15.8 with 4, 16.5 with 16). Past them FULL_CHUNK at least, which pays for a
// workgroup's start (32 sequences up to 4352 in FP16: 36 us with 16, 41 with 8), and about
// WORKGROUPS in all, so that sequences of other lengths than the bound spread evenly
// (64 up to 17920 in 4 bits: 106 us with 2048, 127 with 512, 122 with 8192).
enum { RESIDENT = 512, WORKGROUPS = 2048, MIN_CHUNK = 8, FULL_CHUNK = 16 };

struct AttentionPlan {
    uint32_t tile, tiles, splits, chunk;
};

static AttentionPlan attention_plan(const lh_paged_cache* c, const lh_paged_batch* b,
    uint32_t group)
{
    const uint64_t query = b->max_query < b->tokens ? b->max_query : b->tokens;
    const uint64_t rows = query * group;
    AttentionPlan p;
    p.tile = rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
    const uint64_t tiles = (rows + p.tile - 1) / p.tile;
    p.tiles = (uint32_t)(tiles < 1024 ? tiles : 1024);
    uint64_t longest = (uint64_t)b->table_width * c->page_size;
    longest = b->max_length < longest ? b->max_length : longest;
    const uint64_t steps = (longest + 63) / 64;
    const uint64_t all = tiles * c->kv_heads * b->sequences * steps;
    uint64_t chunk = (all + RESIDENT - 1) / RESIDENT;
    chunk = chunk < MIN_CHUNK ? MIN_CHUNK : chunk;
    if (chunk > FULL_CHUNK) {
        chunk = (all + WORKGROUPS - 1) / WORKGROUPS;
        chunk = chunk < FULL_CHUNK ? FULL_CHUNK : chunk;
    }
    const uint64_t most = 65535 / p.tiles < SPLITS ? 65535 / p.tiles : SPLITS;
    uint64_t splits = (steps + chunk - 1) / chunk;
    splits = splits < most ? splits : most;
    p.splits = (uint32_t)splits;
    p.chunk = (uint32_t)((steps + splits - 1) / splits);
    return p;
}

extern "C" size_t lh_paged_attention_scratch_bytes(const lh_paged_cache* cache,
    const lh_paged_batch* batch, uint32_t group)
{
    const AttentionPlan p = attention_plan(cache, batch, group);
    if (p.splits == 1) {
        return 0;
    }
    return (size_t)batch->tokens * cache->kv_heads * group * p.splits * (cache->head_dim + 2) * 4;
}

template <int D, bool Q4>
static void attention(const lh_paged_cache* c, const lh_paged_batch* b, const AttentionPlan& p,
    const AttentionArgs& a, hipStream_t s)
{
    const dim3 grid(c->kv_heads, b->sequences, p.tiles * p.splits), block(256);
    switch (p.tile) {
    case 4: hipLaunchKernelGGL((k_paged_decode<D, Q4, 4>), grid, block, 0, s, a); break;
    case 8: hipLaunchKernelGGL((k_paged_decode<D, Q4, 8>), grid, block, 0, s, a); break;
    case 16: hipLaunchKernelGGL((k_paged_decode<D, Q4, 16>), grid, block, 0, s, a); break;
    default: hipLaunchKernelGGL((k_paged_attention<D, Q4, 2>), grid, block, 0, s, a); break;
    }
    if (p.splits > 1) {
        const uint32_t query = b->max_query < b->tokens ? b->max_query : b->tokens;
        hipLaunchKernelGGL((k_paged_join<D>), dim3(c->kv_heads * a.group,
            query < 65535 ? query : 65535, b->sequences), block, 0, s, a);
    }
}

extern "C" int lh_launch_paged_attention(const lh_paged_cache* cache, const lh_paged_batch* batch,
    uint32_t group, const float* q, size_t q_stride, float scale, float* out, size_t out_stride,
    uint8_t* scratch, hipStream_t s)
{
    const AttentionPlan p = attention_plan(cache, batch, group);
    const uint32_t in_page = cache->page_size / 32;
    float* part = reinterpret_cast<float*>(scratch);
    float2* tops = reinterpret_cast<float2*>(part + (size_t)batch->tokens * cache->kv_heads *
        group * p.splits * cache->head_dim);
    const AttentionArgs a = {pages_of(cache), batch_of(batch), q, out, part, tops, q_stride,
        out_stride,
        (((uint64_t)1 << 32) + in_page - 1) / in_page, scale * 1.44269504088896341f, group,
        p.splits, p.tiles, p.chunk, p.tile};
    LH_FOR_CACHE(cache, attention, cache, batch, p, a, s);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
