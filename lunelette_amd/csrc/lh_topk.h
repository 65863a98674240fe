// Rows of logits in one pass: the running maximum with the sum of exponentials, and the
// best few tokens, for log probabilities (logprobs.hip) and beams (beam.hip).
#pragma once

#include <type_traits>

#include "lh_device.h"

namespace lh {

// Order of the alternatives as one 64-bit number: the logit's rank (-0 as +0)
// above, the complement of the id below, so a larger key is a likelier token or
// an equal one of lower id. 0 is no token: finite logits have ranks above 0.
__device__ __forceinline__ uint32_t logit_rank(float v)
{
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float rank_logit(uint32_t rank)
{
    return __uint_as_float(rank & 0x80000000u ? rank & 0x7fffffffu : ~rank);
}

__device__ __forceinline__ uint64_t top_key(float v, uint32_t id)
{
    return (uint64_t)logit_rank(v) << 32 | (uint32_t)~id;
}

// Lane l's word of lane l ^ J.
template <int J>
__device__ __forceinline__ uint32_t xor_word(uint32_t v, uint32_t lane)
{
    if (J == 1) {
        return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, false);   // quad_perm [1,0,3,2]
    } else if (J == 2) {
        return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, false);   // quad_perm [2,3,0,1]
    } else if (J == 4) {
        // row_shl:4 into banks 0 and 2, row_shr:4 into banks 1 and 3.
        const uint32_t a = __builtin_amdgcn_update_dpp(0, v, 0x104, 0xf, 0x5, false);
        return __builtin_amdgcn_update_dpp(a, v, 0x114, 0xf, 0xa, false);
    } else if (J == 8) {
        return __builtin_amdgcn_mov_dpp(v, 0x128, 0xf, 0xf, false);  // row_ror:8
    } else if (J == 16) {
        const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return lane & 16 ? p[0] : p[1];
    } else {
        const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return lane & 32 ? p[0] : p[1];
    }
}

// Keeps the larger of the pair (l, l ^ J) where `larger`, the smaller elsewhere.
template <int J>
__device__ __forceinline__ uint64_t exchange(uint64_t key, uint32_t lane, bool larger)
{
    const uint64_t other = (uint64_t)xor_word<J>((uint32_t)(key >> 32), lane) << 32 |
        xor_word<J>((uint32_t)key, lane);
    return (other > key) == larger ? other : key;
}

template <int J>
__device__ __forceinline__ uint64_t half_merge(uint64_t key, uint32_t lane, bool falling)
{
    key = exchange<J>(key, lane, ((lane & J) == 0) == falling);
    if constexpr (J > 1) {
        key = half_merge<J / 2>(key, lane, falling);
    }
    return key;
}

// The 64 lanes' keys in order (bitonic network, 21 exchanges).
__device__ __forceinline__ uint64_t sort_keys(uint64_t key, uint32_t lane, bool falling)
{
    key = half_merge<1>(key, lane, (lane & 2) != 0);
    key = half_merge<2>(key, lane, (lane & 4) != 0);
    key = half_merge<4>(key, lane, (lane & 8) != 0);
    key = half_merge<8>(key, lane, (lane & 16) != 0);
    key = half_merge<16>(key, lane, (lane & 32) != 0);
    return half_merge<32>(key, lane, falling);
}

// The best 64 of `best` (falling) and `rising`, falling.
__device__ __forceinline__ uint64_t merge_best(uint64_t best, uint64_t rising, uint32_t lane)
{
    return half_merge<32>(best > rising ? best : rising, lane, true);
}

// The same network for 32-bit ranks, rising.
template <int J>
__device__ __forceinline__ uint32_t half_merge(uint32_t rank, uint32_t lane, bool falling)
{
    const uint32_t other = xor_word<J>(rank, lane);
    const bool larger = ((lane & J) == 0) == falling;
    rank = larger ? (rank > other ? rank : other) : (rank < other ? rank : other);
    if constexpr (J > 1) {
        rank = half_merge<J / 2>(rank, lane, falling);
    }
    return rank;
}

__device__ __forceinline__ uint32_t sort_ranks(uint32_t rank, uint32_t lane)
{
    rank = half_merge<1>(rank, lane, (lane & 2) != 0);
    rank = half_merge<2>(rank, lane, (lane & 4) != 0);
    rank = half_merge<4>(rank, lane, (lane & 8) != 0);
    rank = half_merge<8>(rank, lane, (lane & 16) != 0);
    rank = half_merge<16>(rank, lane, (lane & 32) != 0);
    return half_merge<32>(rank, lane, false);
}

template <int J>
__device__ __forceinline__ double xor_double(double v, uint32_t lane)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)xor_word<J>((uint32_t)(u >> 32), lane) << 32 |
        xor_word<J>((uint32_t)u, lane));
}

__device__ __forceinline__ double wave_sum(double v, uint32_t lane)
{
    v += xor_double<32>(v, lane);
    v += xor_double<16>(v, lane);
    v += xor_double<8>(v, lane);
    v += xor_double<4>(v, lane);
    v += xor_double<2>(v, lane);
    return v + xor_double<1>(v, lane);
}

// A range of a row: its maximum, the sums relative to it, whether it holds a NaN or
// +Inf.
struct Range {
    double z, w;
    float m;
    uint32_t bad;
};

// The range's sums relative to `to` (no less than its maximum). e^0 is exactly 1.
__device__ __forceinline__ void rescale(Range& r, float to)
{
    if (r.m == -__builtin_inff()) {
        r.z = r.w = 0;
    } else if (r.m != to) {
        const double d = (double)r.m - (double)to, f = exp(d);
        r.w = f * (r.w + d * r.z);
        r.z *= f;
    }
    r.m = to;
}

// e^d for d <= 0: the exponent d log2 e in two parts, the second as a first-order
// factor, so the error is that of the instruction and one rounding.
__device__ __forceinline__ float exp_near(float d)
{
    const float log2e = 1.44269502162933349609375f, rest = 1.92596299112661746887e-8f;
    const float t = d * log2e;
    const float low = __builtin_fmaf(d, rest, __builtin_fmaf(d, log2e, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, low * 0.693147182464599609375f, e);
}

enum { CHUNK = 1024, WAVES = 16, KEYS = 2048 };

// The candidates of a workgroup. The row's chunks deal its logits to 64 groups (the
// lanes); the place `top` among the groups' largest so far bounds the row's from below,
// so those that reach it hold the best `top`, and few others: about 1.5 top in the
// first round of sixteen chunks, ever fewer of a later one.
struct Candidates {
    uint64_t keys[KEYS];
    uint32_t largest[64];   // ranks
    uint32_t count;         // more than KEYS: the row needs the slow way
};

// The bound from the groups' largest; -Inf while fewer than `top` have any. An atomic load,
// which stays a read of LDS: a volatile one waits for the chunks on their way too
// (256 rows of 131072 with 5 alternatives: 1.8 us more).
__device__ __forceinline__ float group_bound(const uint32_t* largest, uint32_t top,
    uint32_t lane)
{
    const uint32_t mine = __hip_atomic_load(&largest[lane], __ATOMIC_RELAXED,
        __HIP_MEMORY_SCOPE_WORKGROUP);
    const uint32_t rank = __builtin_amdgcn_readlane(sort_ranks(mine, lane), 64 - top);
    return rank ? rank_logit(rank) : -__builtin_inff();
}

__device__ __forceinline__ void offer(Candidates& to, float v, uint32_t id, float bound)
{
    if (v >= bound && v > -__builtin_inff()) {
        const uint32_t at = atomicAdd(&to.count, 1u);
        if (at < KEYS) {
            to.keys[at] = top_key(v, id);
        }
    }
}

// The best keys of `live` waves' falling lists, in the first wave. Every wave of the
// workgroup calls it.
__device__ __forceinline__ uint64_t join_lists(uint64_t (&lists)[WAVES][64], uint64_t key,
    uint32_t live, uint32_t wave, uint32_t lane)
{
#pragma unroll 1
    while (live > 1) {
        const uint32_t half = (live + 1) / 2;
        if (wave >= half && wave < live) {
            lists[wave][lane] = key;
        }
        __syncthreads();
        if (wave + half < live) {
            key = merge_best(key, lists[wave + half][63 - lane], lane);
        }
        live = half;
    }
    return key;
}

// Chunk c of a row: lane l has ids 1024 c + 256 q + 4 l + i. Whole chunks load 16 bytes
// a lane, the row's last one looks at every id.
__device__ __forceinline__ void load_chunk(const float* x, uint32_t vocab, uint32_t chunk,
    uint32_t lane, float (&v)[16])
{
    const uint32_t base = chunk * CHUNK + 4 * lane;
    if ((chunk + 1) * CHUNK <= vocab) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float4 f = load4(x + base + 256 * q);
            v[4 * q] = f.x, v[4 * q + 1] = f.y, v[4 * q + 2] = f.z, v[4 * q + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const uint32_t id = base + 256 * (i >> 2) + (i & 3);
            v[i] = x[id < vocab ? id : vocab - 1];
            v[i] = id < vocab ? v[i] : -__builtin_inff();
        }
    }
}

// The best keys of a wave's chunks for rows with more candidates than fit (rising logits,
// many equal ones): the wave keeps a sorted list and sorts every 64 logits into it that
// have one to pass its last place.
__device__ __forceinline__ uint64_t slow_list(const float* x, uint32_t vocab, uint32_t first,
    uint32_t waves, uint32_t top, uint32_t lane)
{
    uint64_t key = 0, least = 0;
#pragma unroll 1
    for (uint32_t at = first; at * CHUNK < vocab; at += waves) {
#pragma unroll 1
        for (uint32_t i = 0; i < CHUNK; i += 64) {
            const uint32_t id = at * CHUNK + i + lane;
            const float v = id < vocab ? x[id] : -__builtin_inff();
            const uint64_t k = v > -__builtin_inff() ? top_key(v, id) : 0;
            if (!__ballot(k > least)) {
                continue;
            }
            key = merge_best(key, sort_keys(k, lane, false), lane);
            least = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), top - 1) << 32 |
                (uint32_t)__builtin_amdgcn_readlane((int)key, top - 1);
        }
    }
    return key;
}

// What the waves of a workgroup share while they scan a part of a row.
struct PartShared {
    Candidates some;
    uint64_t lists[WAVES][64];
    Range ranges[WAVES];
};

// Part `part` of `parts` of a row: its waves take its chunks in turn. To the first wave
// the part's range (in every lane) and its best `top` keys, falling over the lanes.
// WEIGHTED: the sum for the entropy too.
template <bool WEIGHTED>
__device__ __forceinline__ void scan_part(PartShared& sh, const float* x, uint32_t vocab,
    uint32_t top, uint32_t part, uint32_t parts, Range& r, uint64_t& key)
{
    Candidates& some = sh.some;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t chunks = (vocab + CHUNK - 1) / CHUNK, waves = parts * WAVES;
    const uint32_t first = part * WAVES + wave;
    r = {0, 0, -__builtin_inff(), 0};
    float bound = -__builtin_inff();
    bool bad = false;
    float next[16];
    if (first < chunks) {
        load_chunk(x, vocab, first, lane, next);
    }
    if (threadIdx.x < 64) {
        some.largest[threadIdx.x] = 0;
        some.count = 0;
    }
    __syncthreads();
    // first_round: the one in which waves without chunks come for the barrier.
    auto round = [&](uint32_t c, auto first_round) __attribute__((always_inline)) {
        constexpr bool FIRST = decltype(first_round)::value;
        const bool live = !FIRST || c < chunks;
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            v[i] = live ? next[i] : -__builtin_inff();
        }
        if (c + waves < chunks) {
            load_chunk(x, vocab, c + waves, lane, next);
        }
        float four[4], most;   // NaN if any is
#pragma unroll
        for (int q = 0; q < 4; q++) {
            four[q] = __builtin_elementwise_maximum(
                __builtin_elementwise_maximum(v[4 * q], v[4 * q + 1]),
                __builtin_elementwise_maximum(v[4 * q + 2], v[4 * q + 3]));
        }
        most = __builtin_elementwise_maximum(__builtin_elementwise_maximum(four[0], four[1]),
            __builtin_elementwise_maximum(four[2], four[3]));
        // Each lane for itself: in a vote over `most < infinity` the compiler would compare for
        // `not equal` to it, which a NaN passes.
        bad |= !(most < __builtin_inff());
        const bool pass = top && __ballot(most >= bound);
        if (pass && most > -__builtin_inff()) {
            atomicMax(&some.largest[lane], logit_rank(most));
        }
        if (__ballot(most > r.m)) {
            rescale(r, fmaxf(wave_max64(most), r.m));
        }
        const float m = r.m > -__builtin_inff() ? r.m : 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float d = fmaxf(v[i] - m, -150.0f);   // e^-150 is 0, and so is 0 * d
            const float e = exp_near(d);
            r.z += (double)e;
            if (WEIGHTED) {
                r.w += (double)(e * d);
            }
        }
        if (FIRST && top) {
            __syncthreads();   // the groups' largest of the whole first round
        }
        if (pass) {
            bound = group_bound(some.largest, top, lane);
            const uint32_t id = c * CHUNK + 4 * lane;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if (__ballot(four[q] >= bound)) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        offer(some, v[4 * q + i], id + 256 * q + i, bound);
                    }
                }
            }
        }
    };
    round(first, std::true_type());
    for (uint32_t c = first + waves; c < chunks; c += waves) {
        round(c, std::false_type());
    }
    r.bad = __ballot(bad) != 0;
    r.z = wave_sum(r.z, lane);
    if (WEIGHTED) {
        r.w = wave_sum(r.w, lane);
    }
    if (lane == 0) {
        sh.ranges[wave] = r;
    }
    __syncthreads();
    key = 0;
    if (top) {
        // 64 candidates a wave and turn, then the waves' lists.
        uint32_t lists_made = WAVES;
        if (some.count <= KEYS) {
            const uint32_t n = some.count;
            lists_made = (n + 63) / 64 < WAVES ? (n + 63) / 64 : WAVES;
            for (uint32_t i = 64 * wave; i < n; i += 64 * WAVES) {
                const uint64_t mine = i + lane < n ? some.keys[i + lane] : 0;
                key = i < 64 * WAVES ? sort_keys(mine, lane, true)
                    : merge_best(key, sort_keys(mine, lane, false), lane);
            }
        } else {
            key = slow_list(x, vocab, first, waves, top, lane);
        }
        key = join_lists(sh.lists, key, lists_made, wave, lane);
    }
    if (wave) {
        return;
    }
    // Lane w has wave w's range. One more rounding of FP32 for it, where the running
    // maximum's own changes, of which there may be many, take a factor of 64 bits.
    r = lane < WAVES ? sh.ranges[lane] : Range{0, 0, -__builtin_inff(), 0};
    const float to = wave_max64(r.m);
    if (r.m < to) {
        const float d = fmaxf(r.m - to, -150.0f), f = exp_near(d);
        r.w = (double)f * (r.w + (double)d * r.z);
        r.z *= (double)f;
    }
    r.m = to;
    r.z = wave_sum(r.z, lane);
    r.w = wave_sum(r.w, lane);
    r.bad = __ballot(r.bad != 0) != 0;
}

}  // namespace lh
