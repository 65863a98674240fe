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

// The reference of a column's softmax need not be its maximum: it follows once that is
// SLACK (in powers of two) above, so the sums are seldom rescaled (with every new
// maximum some column of a wave has one in most blocks: 59.5 against 56.3 us for 256
// tokens after 4096 positions in 4-bit pages). Probabilities are formed relative to 2^SLACK times the
// reference and stay up to 1 (and a rounding).
//
// The second product takes them (in 4-bit pages times their positions' value scales) times
// a power of two that keeps its planes below 2^15: P_SCALE, or in 4-bit pages one that
// each column lowers when a product of a probability and a scale comes to P_LIMIT. Such a
// product then stands in [2^7, 2^8), and later ones have 2^8 to grow as probabilities
// do. A plane ends at 2^-25: 2^-32 of the largest probability, or product.
constexpr float SLACK = 8, P_SCALE = 32768, P_LIMIT = 32768;

// The power of two that takes a product `most` to [2^7, 2^8), at most `now`.
__device__ __forceinline__ float value_shift(float most, float now)
{
    const int e = (int)((__float_as_uint(most) >> 23) & 0xffu) - 127;
    return fminf(now, exp2i(e < -116 ? 123 : 7 - e));
}

// A column's reference falls by 2^down (<= 0, -Inf for its first): the products so far are
// that much less, so their power of two may rise as much, to 2^123. The factor of their
// sums in the new units.
__device__ __forceinline__ float raise_shift(float& shift, float down)
{
    const uint32_t bits = __float_as_uint(shift);
    const float room = (float)(123 + 127 - (int)(bits >> 23));
    const float up = fminf(-__builtin_floorf(down), room);
    shift = __uint_as_float(bits + ((uint32_t)(int)up << 23));
    return __builtin_amdgcn_exp2f(down + up);
}

// An infinite FP16 value leaves Inf or NaN in its element's sum, by its sign and those of
// the probabilities' planes: NaN it is. (Finite ones cannot overflow: 2^15 * 2^16 each.)
template <bool Q4>
__device__ __forceinline__ float nan_if_odd(float v)
{
    return Q4 ? v : __builtin_fmaf(v, 0.0f, v);
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
// FP16 keys may have an Inf, which has to make the score a NaN: a score of -Inf would be
// left out of the softmax as a hidden position is.
template <int D, bool Q4>
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
    most = column_max(most);
    const int e2 = row_exponent(most);
    const float up = exp2i(e2);
#pragma unroll
    for (int e = 0; e < D / 4; e++) {
        v[e] *= up;
        sum += v[e];
    }
#pragma unroll
    for (int j = 0; j < D / 32; j++) {
        if (Q4) {
            planes8(v + 8 * j, hi[j], lo[j]);
        } else {
            planes8_away(v + 8 * j, hi[j], lo[j]);
        }
    }
    qs = column_sum(sum);
    // Never 0 or Inf, which a hidden or a zero score would turn into NaN. Scores of FP16 keys
    // are below 2^39, so they vanish before cs does; 4-bit keys reach 2^128 and meet cs (to
    // 2^-150), or KEY_UNIT, before the sums, so that any score that FP32 holds is formed. A
    // row of zeros takes the least: its planes may be a step each, and the scale is any.
    cs = most == 0 ? 0x1p-149f : fminf(fmaxf(scale * exp2i(-e2), 0x1p-149f), 3e38f);
}

// Prompts: four waves with 32 query rows each (two column tiles) share every block of 32
// positions in LDS as operands, decoded once by the workgroup: 16 fragments of 64 lanes
// for 128 dims, keys first, and (Q4) the block's scales and zeros as floats.
template <int D, bool Q4>
struct SharedBlock {
    f16x8 fragment[D / 8][64];
    float scale[Q4 ? 4 : 1][32];   // of keys, their zero + 8 scale, of values, theirs
};

template <int D, bool Q4>
struct PromptRows {
    f16x8 hi[2][D / 32], lo[2][D / 32];
    float cs[2], qs[2], m[2], sum[2], offset[2];
    int32_t limit[2], low, high;
    floatx4 acc[2][D / 16];
    float shift[2];   // of the products of probabilities and value scales, a column's own
    bool lost[2];
    uint32_t g, lane;

    __device__ __forceinline__ int32_t position(int32_t base, int e) const
    {
        return base + 4 * (int32_t)g + (e & 3) + 16 * (e >> 2);
    }

    // The scales `which` and their zeros of the lane's positions.
    __device__ __forceinline__ void scales(const SharedBlock<D, Q4>& b, int which,
        float (&scale)[8], float (&z)[8])
    {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const floatx4 x = *reinterpret_cast<const floatx4*>(
                &b.scale[Q4 ? which : 0][16 * t + 4 * g]);
            const floatx4 y = *reinterpret_cast<const floatx4*>(
                &b.scale[Q4 ? which + 1 : 0][16 * t + 4 * g]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                scale[4 * t + i] = x[i];
                z[4 * t + i] = y[i];
            }
        }
    }

    __device__ __forceinline__ void block(const SharedBlock<D, Q4>& b, int32_t base)
    {
        const bool edge = base + 31 > low;
        // Fragments are read a step ahead of their products, and products that need one
        // another stand four apart.
        floatx4 s[2][2];
        f16x8 k[2][2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            k[0][t] = b.fragment[t * (D / 32)][lane];
            s[0][t] = s[1][t] = (floatx4){0, 0, 0, 0};
        }
#pragma unroll
        for (int j = 0; j < D / 32; j++) {
#pragma unroll
            for (int t = 0; t < 2 && j + 1 < D / 32; t++) {
                k[(j + 1) & 1][t] = b.fragment[t * (D / 32) + j + 1][lane];
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int x = 0; x < 4; x++) {
                s[x & 1][x >> 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[j & 1][x >> 1],
                    hi[x & 1][j], s[x & 1][x >> 1], 0, 0, 0);
            }
#pragma unroll
            for (int x = 0; x < 4; x++) {
                s[x & 1][x >> 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[j & 1][x >> 1],
                    lo[x & 1][j], s[x & 1][x >> 1], 0, 0, 0);
            }
        }
        float scale[8], z[8], p[2][8];
        if (Q4) {
            scales(b, 0, scale, z);
        }
#pragma unroll
        for (int n = 0; n < 2; n++) {
            float most;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = s[n][e >> 2][e & 3];
                p[n][e] = Q4 ? __builtin_fmaf(z[e], qs[n], scale[e] * v) : v;
            }
            if (edge) {
                asm volatile("");   // a branch, not selections for every block
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    p[n][e] = position(base, e) > limit[n] ? -__builtin_inff() : p[n][e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                most = e ? fmaxf(most, p[n][e]) : p[n][e];
            }
            most = fmaxf(column_max(most) * cs[n], m[n]);
            if (__ballot(most > m[n] + SLACK)) {
                const float down = m[n] > -__builtin_inff() ? m[n] - most : -__builtin_inff();
                const float keep = __builtin_amdgcn_exp2f(down);
                const float products = Q4 ? raise_shift(shift[n], down) : keep;
                m[n] = most;
                sum[n] *= keep;
                offset[n] *= keep;
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    acc[n][i] *= products;
                }
            }
        }
        if (Q4) {
            scales(b, 2, scale, z);
        }
        f16x8 ph[2], pl[2];
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const float top = (m[n] > -__builtin_inff() ? m[n] : 0.0f) + SLACK;
            float vs[8], vz[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                vs[e] = Q4 ? scale[e] : 0.0f;
                vz[e] = z[e];
            }
            if (Q4 && edge) {
                asm volatile("");
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const bool hidden = position(base, e) > limit[n];
                    vs[e] = hidden ? 0.0f : vs[e];   // may hold anything
                    vz[e] = hidden ? 0.0f : vz[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                p[n][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[n][e], cs[n], -top));
                sum[n] += p[n][e];
                if (Q4) {
                    offset[n] = __builtin_fmaf(p[n][e], vz[e], offset[n]);
                    p[n][e] *= vs[e];
                } else {
                    p[n][e] *= P_SCALE;
                }
            }
            if (Q4) {
                float most = p[n][0];
#pragma unroll
                for (int e = 1; e < 8; e++) {
                    most = fmaxf(most, p[n][e]);
                }
                if (__ballot(most * shift[n] >= P_LIMIT)) {
                    const float next = value_shift(column_max(most), shift[n]);
                    const float ratio = next / shift[n];
#pragma unroll
                    for (int i = 0; i < D / 16; i++) {
                        acc[n][i] *= ratio;
                    }
                    shift[n] = next;
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    p[n][e] *= shift[n];
                }
            }
            planes8(p[n], ph[n], pl[n]);
        }
        f16x8 v[2][2];
#pragma unroll
        for (int x = 0; x < 2; x++) {
            v[0][x] = b.fragment[D / 16 + x][lane];
        }
#pragma unroll
        for (int i = 0; i < D / 16; i += 2) {
            const int at = (i / 2) & 1;
#pragma unroll
            for (int x = 0; x < 2 && i + 2 < D / 16; x++) {
                v[at ^ 1][x] = b.fragment[D / 16 + i + 2 + x][lane];
            }
            __builtin_amdgcn_sched_barrier(0);
            if (!Q4 && edge) {
                v[at][0] = without_odd(v[at][0], i, base);
                v[at][1] = without_odd(v[at][1], i + 1, base);
            }
#pragma unroll
            for (int x = 0; x < 4; x++) {
                acc[x & 1][i + (x >> 1)] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[at][x >> 1],
                    ph[x & 1], acc[x & 1][i + (x >> 1)], 0, 0, 0);
            }
#pragma unroll
            for (int x = 0; x < 4; x++) {
                acc[x & 1][i + (x >> 1)] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[at][x >> 1],
                    pl[x & 1], acc[x & 1][i + (x >> 1)], 0, 0, 0);
            }
        }
    }

    // v with every Inf or NaN as 0: it may stand at a position that some row does not see,
    // or that holds no value yet. Rows that see it get NaN.
    __device__ __forceinline__ f16x8 without_odd(f16x8 v, int i, int32_t base)
    {
        f16x8 odd;
        bool any = false;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const bool bad = !__builtin_isfinite((float)v[e]);
            odd[e] = bad && position(base, e) <= high ? (_Float16)1 : (_Float16)0;
            any |= bad && position(base, e) <= high;
            v[e] = bad ? (_Float16)0 : v[e];
        }
        if (__ballot(any)) {
#pragma unroll
            for (int n = 0; n < 2; n++) {
                f16x8 on;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    on[e] = position(base, e) <= limit[n] ? (_Float16)1 : (_Float16)0;
                }
                const floatx4 hits = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, on,
                    (floatx4){0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    acc[n][i][r] = hits[r] > 0 ? __builtin_nanf("") : acc[n][i][r];
                }
            }
        }
        return v;
    }
};

// Of the scales and zeros of a prompt's 4-bit keys in LDS: with keys up to 2^128 their
// products with a query's sums (up to 2^25) stay in FP32's range, and keys count to 2^-125.
// (Meeting cs before the sums, as in the decode kernel, takes 32 instructions a block here:
// 55.9 against 55.1 us for 256 tokens after 4096.)
constexpr float KEY_UNIT = 0x1p-24f;

enum { PROMPT_ROWS = 128 };

// grid (KV heads, sequences, tiles of the splits in turn): the tiles of a KV head of
// eight share an XCD and its L2. One barrier a block: while a block is multiplied the
// next one is decoded into the other buffer and the one after is on its way.
// Of 4-bit pages two teams of four waves take every second block of a split for the same
// rows and meet in LDS at its end, which halves the parts that splits leave in memory (256
// tokens after 4096: 56.3 us, with one team and twice the workgroups 59.1; 64 tokens 30.8
// and 36.3). FP16 pages wait for the other team's loads too then (256 tokens: 56.5
// against 54.5, though 64 tokens 31.6 against 35.9).
template <bool Q4>
constexpr int TEAMS = Q4 ? 2 : 1;

template <int D, bool Q4>
__global__ void __launch_bounds__(256 * TEAMS<Q4>, 2)
k_paged_prompt(AttentionArgs a)
{
    typedef PageLayout<D, Q4> Layout;
    constexpr int STEP = TEAMS<Q4>;
    constexpr uint32_t LOADERS = D / 32;   // waves that bring four fragments each
    __shared__ SharedBlock<D, Q4> buffers[2 * STEP];
    __shared__ float stats[4][2][2][16];   // of the second team: [wave][column tile][m, sum]
    const uint32_t h = blockIdx.x, s = blockIdx.y, lane = threadIdx.x & 63;
    const uint32_t waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t team = STEP > 1 ? waves >> 2 : 0, wave = STEP > 1 ? waves & 3 : waves;
    SharedBlock<D, Q4>* blocks = buffers + 2 * team;
    const uint32_t split = blockIdx.z / a.tiles;
    const Span span = batch_span(a.batch, s);
    const int64_t rows = span.count * a.group;
    const int64_t capacity = (int64_t)a.batch.width * a.cache.page_size;
    const uint32_t in_page = a.cache.page_size / 32;
    const int32_t* table = a.batch.table + (size_t)s * a.batch.width;
    const size_t head_bytes = Layout::head_bytes(a.cache.page_size);
    const NibbleMasks mask;
    for (int64_t tile = blockIdx.z % a.tiles; tile * PROMPT_ROWS < rows; tile += a.tiles) {
        auto limit_of = [&](int64_t row) __attribute__((always_inline)) {
            const int64_t last = span.first + row / a.group;
            return last < 0 ? -1 : (int32_t)(last < capacity ? last : capacity - 1);
        };
        const int64_t last_row = tile * PROMPT_ROWS + PROMPT_ROWS < rows
            ? tile * PROMPT_ROWS + PROMPT_ROWS - 1 : rows - 1;
        const int32_t high = limit_of(last_row);
        const int32_t steps = high < 0 ? 0 : (high >> 6) + 1, all = high < 0 ? 0 : (high >> 5) + 1;
        const int32_t chunk = split_chunk(a, steps);
        if (split && (int64_t)split * chunk >= steps) {
            continue;   // nothing for this split: the join does not ask for it
        }
        const int32_t start = 2 * (int32_t)split * chunk, first = start + (int32_t)team;
        const int32_t end = all - start < 2 * chunk ? all : start + 2 * chunk;
        PromptRows<D, Q4> c;
        c.lane = lane;
        c.g = lane >> 4;
        // Lane i has the page ids of the team's blocks 64 n + i.
        int32_t ids = 0;
        u32x4 raw;
        uint32_t words = 0;
        bool good = true;
        auto locate = [&](int32_t b, uint32_t& slot) __attribute__((always_inline)) {
            const int32_t turn = (b - first) / STEP;
            if ((turn & 63) == 0) {
                const uint64_t block = (uint32_t)b + STEP * lane;
                const int64_t at = (int64_t)(block * a.per_page >> 32);
                ids = at < a.batch.width ? table[at] : -1;
            }
            const uint32_t page = (uint32_t)((uint64_t)(uint32_t)b * a.per_page >> 32);
            int32_t id = __builtin_amdgcn_readlane(ids, turn & 63);
            good = id >= 0 && (uint32_t)id < a.cache.pages;
            slot = 32 * ((uint32_t)b - page * in_page);
            // A block without a place reads page 0 and is lost for the rows that see it.
            return a.cache.base + ((size_t)(good ? id : 0) * a.cache.kv_heads + h) * head_bytes;
        };
        auto missing = [&](int32_t b) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < 2; n++) {
                c.lost[n] |= !good && 32 * b <= c.limit[n];
            }
        };
        // Q4: asks for block b's words.
        auto ask = [&](int32_t b) __attribute__((always_inline)) {
            uint32_t slot;
            const uint8_t* part = locate(b, slot);
            missing(b);
            const uint8_t* key = part + slot * Layout::vector;
            const uint8_t* value = key + Layout::values(a.cache.page_size);
            if (wave < LOADERS / 2) {
                if (D == 64) {
                    const uint2 x = reinterpret_cast<const uint2*>(key)[lane];
                    const uint2 y = reinterpret_cast<const uint2*>(key)[64 + lane];
                    raw = (u32x4){x.x, x.y, y.x, y.y};
                } else {
                    raw = reinterpret_cast<const u32x4*>(key)[64 * wave + lane];
                }
            } else if (wave < LOADERS) {
                raw = reinterpret_cast<const u32x4*>(value)[64 * (wave - LOADERS / 2) + lane];
            }
            if (wave == 0) {
                words = *reinterpret_cast<const uint32_t*>(part +
                    Layout::scales(a.cache.page_size, lane >> 5) + 4 * (slot + (lane & 31)));
            }
        };
        // Q4: block b, asked for before, into `to`.
        auto decode = [&](int32_t b, SharedBlock<D, Q4>& to) __attribute__((always_inline)) {
            if (wave < LOADERS) {
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    to.fragment[4 * wave + w][lane] = codes_minus8(raw[w], mask);
                }
            }
            if (wave == 0) {
                const float unit = lane < 32 ? KEY_UNIT : 1.0f;
                float scale = bf16_to_f32(words & 0xffffu) * unit;
                float z = __builtin_fmaf(8.0f, scale,
                    __uint_as_float(words & 0xffff0000u) * unit);
                if (32 * b + (int32_t)(lane & 31) > high) {
                    scale = z = 0;   // may hold anything
                }
                to.scale[Q4 ? 2 * (lane >> 5) : 0][lane & 31] = scale;
                to.scale[Q4 ? 2 * (lane >> 5) + 1 : 0][lane & 31] = z;
            }
        };
        // F16: block b straight into `to`.
        auto fetch = [&](int32_t b, SharedBlock<D, Q4>& to) __attribute__((always_inline)) {
            uint32_t slot;
            const uint8_t* part = locate(b, slot);
            missing(b);
            const uint8_t* key = part + slot * Layout::vector;
            const uint8_t* value = key + Layout::values(a.cache.page_size);
            if (wave < LOADERS) {
                const uint8_t* from = wave < LOADERS / 2 ? key + 4096 * wave
                    : value + 4096 * (wave - LOADERS / 2);
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    __builtin_amdgcn_global_load_lds(
                        (const __attribute__((address_space(1))) void*)(from + 1024 * w +
                            16 * lane),
                        (__attribute__((address_space(3))) void*)&to.fragment[4 * wave + w][0], 16,
                        0, 0);
                }
            }
        };
        // Rows past the last one repeat it and are not stored.
        auto row_of = [&](int n) __attribute__((always_inline)) {
            const int64_t row = tile * PROMPT_ROWS + 32 * wave + 16 * n + (lane & 15);
            return row < rows ? row : rows - 1;
        };
#pragma unroll
        for (int n = 0; n < 2; n++) {
            c.lost[n] = span.first + row_of(n) / a.group >= capacity;
            c.limit[n] = limit_of(row_of(n));
            c.m[n] = -__builtin_inff();
            c.sum[n] = c.offset[n] = 0;
            c.shift[n] = exp2i(123);
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                c.acc[n][i] = (floatx4){0, 0, 0, 0};
            }
        }
        // Limits do not fall from a row to the next.
        c.low = __builtin_amdgcn_readlane(c.limit[0], 0);
        c.high = __builtin_amdgcn_readlane(c.limit[1], 15);
        __syncthreads();   // the previous tile's readers
        if (first < end) {
            if constexpr (Q4) {
                ask(first);
            } else {
                fetch(first, blocks[0]);
            }
        }
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const int64_t row = row_of(n);
            load_query<D, Q4>(a.q + (size_t)(span.begin + row / a.group) * a.q_stride +
                ((size_t)h * a.group + row % a.group) * D, c.g, a.scale, c.hi[n], c.lo[n], c.cs[n],
                c.qs[n]);
            if (Q4) {
                c.cs[n] = fminf(c.cs[n] / KEY_UNIT, 3e38f);
            }
        }
        if (Q4 && first < end) {
            decode(first, blocks[0]);
            if (first + STEP < end) {
                ask(first + STEP);
            }
        }
        // Both teams pass the same barriers.
        for (int32_t b = first; b - (int32_t)team < end; b += STEP) {
            const int32_t turn = (b - first) / STEP & 1;
            SharedBlock<D, Q4>&now = blocks[turn], &other = blocks[1 - turn];
            if (!Q4) {
                __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): this wave's part of the block
            }
            __syncthreads();   // this block is there, the other buffer is free
            if (b + STEP < end) {
                if constexpr (Q4) {
                    decode(b + STEP, other);
                    if (b + 2 * STEP < end) {
                        ask(b + 2 * STEP);
                    }
                } else {
                    fetch(b + STEP, other);
                }
            }
            if (b < end && 32 * b <= c.high) {
                c.block(now, 32 * b);
            }
        }
        // The second team's sums, relative to its own maxima, to the first.
        if (STEP > 1) {
            __syncthreads();
        }
        floatx4* joined = reinterpret_cast<floatx4*>(buffers) + wave * (D / 8) * 64 + lane;
        float sum[2];
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const float back = Q4 ? 1.0f / c.shift[n] : 1.0f / P_SCALE;   // powers of two
            sum[n] = c.lost[n] ? __builtin_nanf("") : column_sum(c.sum[n]);
            const float offset = Q4 ? column_sum(c.offset[n]) : 0.0f;
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    c.acc[n][i][r] = nan_if_odd<Q4>(
                        __builtin_fmaf(c.acc[n][i][r], back, offset));
                }
                if (team) {
                    joined[(n * (D / 16) + i) * 64] = c.acc[n][i];
                }
            }
            if (team && c.g == 0) {
                stats[wave][n][0][lane] = c.m[n];
                stats[wave][n][1][lane] = sum[n];
            }
        }
        if (STEP > 1) {
            __syncthreads();
        }
        if (team) {
            continue;   // its next tile begins with a barrier, before LDS is written again
        }
        const bool whole = steps <= chunk;   // no other split has a part
#pragma unroll
        for (int n = 0; n < 2; n++) {
            if (tile * PROMPT_ROWS + 32 * wave + 16 * n + (lane & 15) >= rows) {
                continue;
            }
            // A team that saw nothing holds sums of 0, or NaN for a lost position.
            float m = c.m[n], keep = 1, keep1 = 0, all_sum = sum[n];
            if (STEP > 1) {
                const float m1 = stats[wave][n][0][lane & 15];
                m = fmaxf(m, m1);
                keep = c.m[n] > -__builtin_inff() ? __builtin_amdgcn_exp2f(c.m[n] - m) : 1.0f;
                keep1 = m1 > -__builtin_inff() ? __builtin_amdgcn_exp2f(m1 - m) : 1.0f;
                all_sum = __builtin_fmaf(stats[wave][n][1][lane & 15], keep1, sum[n] * keep);
            }
            // (No position at all: 0.)
            const float over = whole ? all_sum == 0 ? 0.0f : 1.0f / all_sum : 1.0f;
            const int64_t row = row_of(n);
            const size_t token = (size_t)(span.begin + row / a.group);
            const size_t head = (size_t)h * a.group + row % a.group;
            const size_t at = (token * a.cache.kv_heads * a.group + head) * a.splits + split;
            float* to = whole ? a.out + token * a.out_stride + head * D : a.part + at * D;
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                floatx4 y = c.acc[n][i];
                if (STEP > 1) {
                    const floatx4 other = joined[(n * (D / 16) + i) * 64];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        y[r] = __builtin_fmaf(other[r], keep1, y[r] * keep);
                    }
                }
                const float4 v = make_float4(y[0] * over, y[1] * over, y[2] * over, y[3] * over);
                store4(to + 16 * i + 4 * c.g, v);
            }
            if (!whole && c.g == 0) {
                a.tops[at] = make_float2(m, all_sum);
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

    // Scores of the lane's positions, of FP16 keys in units of 1 / cs.
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
        }
        // Products that need one another stand four apart.
#pragma unroll
        for (int j = 0; j < D / 32; j++) {
            const f16x8 qh = SHARED ? planes[64 * j + at] : hi[SHARED ? 0 : j];
            const f16x8 ql = SHARED ? planes[64 * (D / 32 + j) + at] : lo[SHARED ? 0 : j];
            f16x8 x[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int w = (t & 1) * (D / 32) + j;
                x[t] = Q4 ? codes_minus8(step.k[t >> 1][w >> 2][w & 3], mask)
                    : __builtin_bit_cast(f16x8, step.k[t >> 1][Q4 ? 0 : w]);
            }
#pragma unroll
            for (int t = 0; t < 4; t++) {
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[t], qh, s[t], 0, 0, 0);
            }
#pragma unroll
            for (int t = 0; t < 4; t++) {
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[t], ql, s[t], 0, 0, 0);
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
                    y = __builtin_fmaf(z * cs, qs, scale * cs * y);
                }
                p[4 * w + i] = y;
            }
        }
    }

    // The softmax over the step and the operands of the second product: p (times the
    // value scales) in planes, pairs 0 and 1 of tile PACK * w + u in words 2 w and 2 w + 1.
    __device__ __forceinline__ void probabilities(const Step& step, float (&p)[C], int32_t base,
        bool edge, uint32_t (&ph)[C / 2], uint32_t (&pl)[C / 2])
    {
        float scale[C], z[C];
        if (Q4) {
#pragma unroll
            for (int e = 0; e < C; e++) {
                const uint32_t word = step.vs[e >> 2][e & 3];
                scale[e] = bf16_to_f32(word & 0xffffu);
                z[e] = __builtin_fmaf(8.0f, scale[e], __uint_as_float(word & 0xffff0000u));
                if (edge && position(base, e) > limit) {
                    scale[e] = z[e] = 0;   // may hold anything
                }
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
        most = fmaxf(Q4 ? column_max(most) : column_max(most) * cs, m);
        if (__ballot(most > m + SLACK)) {
            const float down = m > -__builtin_inff() ? m - most : -__builtin_inff();
            const float keep = __builtin_amdgcn_exp2f(down);
            const float products = Q4 ? raise_shift(shift, down) : keep;
            m = most;
            sum *= keep;
            offset *= keep;
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                acc[i] *= products;
            }
        }
        const float top = (m > -__builtin_inff() ? m : 0.0f) + SLACK;
#pragma unroll
        for (int e = 0; e < C; e++) {
            p[e] = __builtin_amdgcn_exp2f(Q4 ? p[e] - top : __builtin_fmaf(p[e], cs, -top));
            sum += p[e];
            if (Q4) {
                offset = __builtin_fmaf(p[e], z[e], offset);
                p[e] *= scale[e];
            } else {
                p[e] *= P_SCALE;
            }
        }
        if (Q4) {
            most = p[0];
#pragma unroll
            for (int e = 1; e < C; e++) {
                most = fmaxf(most, p[e]);
            }
            if (__ballot(most * shift >= P_LIMIT)) {
                const float next = value_shift(column_max(most), shift), ratio = next / shift;
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    acc[i] *= ratio;
                }
                shift = next;
            }
#pragma unroll
            for (int e = 0; e < C; e++) {
                p[e] *= shift;
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
        auto keys = [&](auto& to) __attribute__((always_inline)) {
            to.load_keys(part, slot, a.cache.page_size, lane);
        };
        auto values = [&](auto& to) __attribute__((always_inline)) {
            to.load_values(part, slot, a.cache.page_size, lane);
        };
        if (x < end) {
            locate(x, 0);
            keys(step);
            values(step);
        }
        const float* q = a.q + (size_t)(span.begin + t) * a.q_stride +
            ((size_t)h * a.group + row % a.group) * D;
        if constexpr (Decode<D, Q4, C>::SHARED) {
            f16x8 hi[D / 32], lo[D / 32];
            load_query<D, Q4>(q, c.g, a.scale, hi, lo, c.cs, c.qs);
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
            load_query<D, Q4>(q, c.g, a.scale, c.hi, c.lo, c.cs, c.qs);
        }
        int32_t turn = 0;
        if constexpr (Q4) {
            // A step is little: the next one's loads run during all of this one (the last
            // one asks for itself again, which spares every step a selection).
            while (x < end) {
                const int32_t base = 64 * x;
                const bool edge = base + 63 > c.low, more = x + 4 < end;
                float p[C];
                uint32_t ph[C / 2], pl[C / 2];
                DecodeStep<D, Q4, C> next;
                turn += more ? 1 : 0;
                locate(more ? x + 4 : x, turn);
                keys(next);
                values(next);
                x += 4;
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
        const float back = keep * (Q4 ? 1.0f / c.shift : 1.0f / P_SCALE);   // powers of two
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            floatx4 y;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                y[r] = nan_if_odd<Q4>(
                    __builtin_fmaf(c.acc[i][r], back, Q4 ? c.offset * keep : 0.0f));
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

// The splits that the tile of row (t, head) had: nothing to join at one.
__device__ __forceinline__ uint32_t join_splits(const AttentionArgs& a, const Span& span,
    int64_t t, uint32_t head)
{
    const int64_t rows = span.count * a.group;
    const int64_t capacity = (int64_t)a.batch.width * a.cache.page_size;
    int64_t end = (t * a.group + head % a.group) / a.tile * a.tile + a.tile;
    end = end < rows ? end : rows;
    int64_t last = span.first + (end - 1) / a.group;
    last = last < capacity ? last : capacity - 1;
    const int32_t steps = last < 0 ? 0 : (int32_t)(last >> 6) + 1;
    const int32_t chunk = split_chunk(a, steps);
    return steps <= chunk ? 1 : (uint32_t)((steps + chunk - 1) / chunk);
}

// Joins up to FEW_SPLITS splits: D / 4 threads a row, all parts asked for at once.
enum { FEW_SPLITS = 8 };

template <int D>
__global__ void __launch_bounds__(256)
k_paged_join_few(AttentionArgs a)
{
    constexpr uint32_t QUADS = D / 4, EACH = 256 / QUADS;
    const uint32_t s = blockIdx.y, heads = a.cache.kv_heads * a.group;
    const uint32_t quad = threadIdx.x % QUADS;
    const Span span = batch_span(a.batch, s);
    for (int64_t i = (int64_t)blockIdx.x * EACH + threadIdx.x / QUADS; i < span.count * heads;
         i += (int64_t)gridDim.x * EACH) {
        const int64_t t = i / heads;
        const uint32_t head = (uint32_t)(i % heads);
        const uint32_t splits = join_splits(a, span, t, head);
        if (splits == 1) {
            continue;   // written already
        }
        const size_t token = (size_t)(span.begin + t), row = (token * heads + head) * a.splits;
        float2 tops[FEW_SPLITS];
        float4 part[FEW_SPLITS];
        float m = -__builtin_inff(), sum = 0;
        float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
        for (uint32_t x = 0; x < FEW_SPLITS; x++) {
            const uint32_t at = x < splits ? x : splits - 1;
            tops[x] = a.tops[row + at];
            part[x] = reinterpret_cast<const float4*>(a.part)[(row + at) * QUADS + quad];
            m = fmaxf(m, tops[x].x);
        }
#pragma unroll
        for (uint32_t x = 0; x < FEW_SPLITS; x++) {
            // A split that saw nothing holds sums of 0, or NaN for a lost position.
            float keep = tops[x].x > -__builtin_inff() ? __builtin_amdgcn_exp2f(tops[x].x - m)
                : 1.0f;
            if (x >= splits) {
                continue;
            }
            sum = __builtin_fmaf(tops[x].y, keep, sum);
            v.x = __builtin_fmaf(part[x].x, keep, v.x);
            v.y = __builtin_fmaf(part[x].y, keep, v.y);
            v.z = __builtin_fmaf(part[x].z, keep, v.z);
            v.w = __builtin_fmaf(part[x].w, keep, v.w);
        }
        const float over = sum == 0 ? 0.0f : 1.0f / sum;
        store4(a.out + token * a.out_stride + (size_t)head * D + 4 * quad,
            make_float4(v.x * over, v.y * over, v.z * over, v.w * over));
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
    for (int64_t t = blockIdx.y; t < span.count; t += gridDim.y) {
        const uint32_t splits = join_splits(a, span, t, head);
        if (splits == 1) {
            continue;   // written already
        }
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

// How the steps are split. RESIDENT workgroups of the tiles of 4 and 8 rows are on the chip
// at once (of the tiles of 16 rows of 128 dims, one wave a SIMD, half as many, which the
// plan does not go by); up to them a split takes as few as MIN_CHUNK steps (one sequence
// of 15999 positions: 13.9 us with 8, 16.5 with 4, 15.2 with 12). Past them FULL_CHUNK at
// least, which pays for a workgroup's start (32 sequences up to 4352 in FP16: 36.1 us,
// with 12 36.5, with 24 44.1), and about WORKGROUPS in all, so that sequences of other
// lengths than the bound spread evenly (64 up to 17920 in 4 bits: 102 us with 2048, 99
// with 1024, 121 with 512, 118 with 8192; in FP16 285, 328, 313 and 289).
// A prompt's workgroup (team) has 128 rows, and the splits' parts are as large as its
// output for each: PROMPT_WORKGROUPS teams in all (256 tokens after 4096 positions in 4-bit
// pages: 56.3 us with 512, 86.6 with 256, 70.0 with 1024; FP16 54.5, 61.4 and 76.1),
// PROMPT_CHUNK steps at least.
enum { RESIDENT = 512, WORKGROUPS = 2048, MIN_CHUNK = 8, FULL_CHUNK = 16,
    PROMPT_WORKGROUPS = 512, PROMPT_CHUNK = 4 };

struct AttentionPlan {
    uint32_t tile, tiles, splits, chunk;
};

static AttentionPlan attention_plan(const lh_paged_cache* c, const lh_paged_batch* b,
    uint32_t group)
{
    const uint64_t query = b->max_query < b->tokens ? b->max_query : b->tokens;
    const uint64_t rows = query * group;
    AttentionPlan p;
    // The least tile that has all rows of a sequence, to 32 (8 sequences of 500 to 4352 in 4
    // bits and in FP16, group 4: up to 4 tokens each take 28.5 and 33.3 us, with the
    // prompts' tile 47.8 and 43.5; up to 8 take 33.9 and 37.5 against 48.2 and 43.9; up to
    // 16 take 48.3 and 53.5 with tiles of 16 rows, 49.5 and 45.8 with the prompts').
    p.tile = rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 32 ? 16 : PROMPT_ROWS;
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
    if (p.tile == PROMPT_ROWS) {
        const uint32_t groups = PROMPT_WORKGROUPS / (c->kind == LH_CACHE_Q4 ? TEAMS<true> : 1);
        chunk = (all + groups - 1) / groups;
        chunk = chunk < PROMPT_CHUNK ? PROMPT_CHUNK : chunk;
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
    default: hipLaunchKernelGGL((k_paged_prompt<D, Q4>), grid, dim3(256 * TEAMS<Q4>), 0, s, a);
        break;
    }
    if (p.splits > 1) {
        const uint32_t query = b->max_query < b->tokens ? b->max_query : b->tokens;
        const uint64_t each = (uint64_t)query * c->kv_heads * a.group * D / 1024;
        if (p.splits <= FEW_SPLITS) {
            hipLaunchKernelGGL((k_paged_join_few<D>), dim3(each < 1 ? 1 : each > 4096 ? 4096 : each,
                b->sequences), block, 0, s, a);
            return;
        }
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
    return (int)hipGetLastError();
}
