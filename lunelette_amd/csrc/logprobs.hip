// Log probabilities, entropy and top alternatives of logit rows (lh_logprobs).
//
// With m = max x and Z = sum e^(x - m): ln p_t = (x_t - m) - ln Z and
// H = ln Z - sum e^(x - m) (x - m) / Z. Both are sums of terms of one sign, so
// nothing cancels; the sums run in 64 bits (as fast as 32 on this chip) and the
// largest logit's own term is exactly 1, so where one token has nearly all the
// probability ln Z keeps the relative precision of the other terms. Each of those is
// off by |x - m| 2^-24 of itself (x - m is rounded to FP32 before the exponential) and
// the exponential's two steps: 1e-6 at a distance of 20.
//
// One pass: a row is dealt to workgroups (one or more a row), each wave reads chunks
// of 1024 logits with the running maximum and the two sums and puts the few that may
// be among the best `top` aside; both meet in the workgroup and, where a row has more
// than one, in a second launch. Bound by the reads: 256 rows of 131072 with 5 alternatives
// 31 us, 4.4 TB/s (28 us without any, 21 us for a plain read of as much); one row is
// two launches and their memory round trips, 12 us.
#include "lh_device.h"
#include "lh_serving.h"

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

__device__ __forceinline__ double wave_sum(double v)
{
    for (int s = 32; s; s >>= 1) {
        v += __shfl_xor(v, s);
    }
    return v;
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

enum { CHUNK = 1024, WAVES = 16, KEYS = 2048, LOGPROB_PARTS = 64 };

// The candidates of a workgroup. The row's chunks deal its logits to 64 groups (the
// lanes); the place `top` among the groups' largest so far bounds the row's from below,
// so those that reach it hold the best `top`, and few others: about 1.5 top in the
// first round of sixteen chunks, ever fewer of a later one.
struct Candidates {
    uint64_t keys[KEYS];
    uint32_t largest[64];   // ranks
    uint32_t count;         // more than KEYS: the row needs the slow way
};

// The bound from the groups' largest; -Inf while fewer than `top` have any.
__device__ __forceinline__ float group_bound(const volatile uint32_t* largest, uint32_t top,
    uint32_t lane)
{
    const uint32_t rank = __builtin_amdgcn_readlane(sort_ranks(largest[lane], lane), 64 - top);
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

struct LogprobArgs {
    const float* logits;
    const int64_t* tokens;
    float *logprob, *entropy, *top_logprobs;
    int64_t* top_ids;
    Range* ranges;      // [row][part]
    uint64_t* keys;     // [row][part][top]
    size_t stride;
    uint32_t vocab, top, parts;
};

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

// Outputs of a row from its whole range and (in the first wave's lanes) its best keys.
__device__ __forceinline__ void finish(const LogprobArgs& a, size_t row, const Range& r,
    uint64_t key, uint32_t lane)
{
    const bool bad = r.bad, empty = r.m == -__builtin_inff();
    const double log_z = log(r.z);
    const float nan = __builtin_nanf("");
    if (lane == 0 && a.logprob) {
        const int64_t t = a.tokens[row];
        float v = nan;
        if (t == -1 && !bad) {
            v = 0;
        } else if (t >= 0 && t < (int64_t)a.vocab && !bad) {
            v = empty ? -__builtin_inff()
                : (float)((double)a.logits[row * a.stride + t] - (double)r.m - log_z);
        }
        a.logprob[row] = v;
    }
    if (lane == 0 && a.entropy) {
        a.entropy[row] = bad ? nan : empty ? 0.0f : (float)(log_z - r.w / r.z);
    }
    if (lane < a.top) {
        const bool none = bad || !key;
        a.top_ids[row * a.top + lane] = none ? -1 : (int64_t)(uint32_t)~(uint32_t)key;
        a.top_logprobs[row * a.top + lane] = bad ? nan : !key ? -__builtin_inff()
            : (float)((double)rank_logit((uint32_t)(key >> 32)) - (double)r.m - log_z);
    }
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

// grid (parts, rows). The waves of a part take its chunks in turn.
__global__ void __launch_bounds__(64 * WAVES)
k_logprob_ranges(LogprobArgs a)
{
    __shared__ Candidates some;
    __shared__ uint64_t lists[WAVES][64];
    __shared__ Range ranges[WAVES];
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const size_t row = blockIdx.y;
    const float* x = a.logits + row * a.stride;
    const uint32_t chunks = (a.vocab + CHUNK - 1) / CHUNK, waves = a.parts * WAVES;
    const uint32_t first = blockIdx.x * WAVES + wave;
    Range r = {0, 0, -__builtin_inff(), 0};
    float bound = -__builtin_inff();
    bool bad = false;
    float next[16];
    if (first < chunks) {
        load_chunk(x, a.vocab, first, lane, next);
    }
    if (threadIdx.x < 64) {
        some.largest[threadIdx.x] = 0;
        some.count = 0;
    }
    __syncthreads();
    for (uint32_t c = first; c < chunks || c == first; c += waves) {
        const bool live = c < chunks;   // a wave without chunks comes for the barrier
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            v[i] = live ? next[i] : -__builtin_inff();
        }
        if (c + waves < chunks) {
            load_chunk(x, a.vocab, c + waves, lane, next);
        }
        float most = v[0];   // NaN if any is
#pragma unroll
        for (int i = 1; i < 16; i++) {
            most = __builtin_elementwise_maximum(most, v[i]);
        }
        bad |= !(most < __builtin_inff());
        const bool pass = a.top && __ballot(most >= bound);
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
            r.w += (double)(e * d);
        }
        if (c == first && a.top) {
            __syncthreads();   // the groups' largest of the whole first round
        }
        if (pass) {
            bound = group_bound(some.largest, a.top, lane);
            const uint32_t id = c * CHUNK + 4 * lane;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                offer(some, v[i], id + 256 * (i >> 2) + (i & 3), bound);
            }
        }
    }
    r.bad = __ballot(bad) != 0;
    r.z = wave_sum(r.z);
    r.w = wave_sum(r.w);
    if (lane == 0) {
        ranges[wave] = r;
    }
    __syncthreads();
    uint64_t key = 0;
    if (a.top) {
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
            key = slow_list(x, a.vocab, first, waves, a.top, lane);
        }
        key = join_lists(lists, key, lists_made, wave, lane);
    }
    if (wave) {
        return;
    }
    // Lane w has wave w's range. One more rounding of FP32 for it, where the running
    // maximum's own changes, of which there may be many, take a factor of 64 bits.
    r = lane < WAVES ? ranges[lane] : Range{0, 0, -__builtin_inff(), 0};
    const float to = wave_max64(r.m);
    if (r.m < to) {
        const float d = fmaxf(r.m - to, -150.0f), f = exp_near(d);
        r.w = (double)f * (r.w + (double)d * r.z);
        r.z *= (double)f;
    }
    r.m = to;
    r.z = wave_sum(r.z);
    r.w = wave_sum(r.w);
    r.bad = __ballot(r.bad != 0) != 0;
    if (a.parts == 1) {
        finish(a, row, r, key, lane);
        return;
    }
    const size_t at = row * a.parts + blockIdx.x;
    if (lane == 0) {
        a.ranges[at] = r;
    }
    if (lane < a.top) {
        a.keys[at * a.top + lane] = key;
    }
}

// Joins a row's parts (at most 64): lane p of the first wave has part p's range; sixteen
// waves take four parts' keys each, all asked for at once, and halve the lists.
__global__ void __launch_bounds__(64 * WAVES)
k_logprob_join(LogprobArgs a)
{
    __shared__ uint64_t lists[WAVES][64];
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const size_t row = blockIdx.x;
    Range r = {0, 0, -__builtin_inff(), 0};
    if (wave == 0 && lane < a.parts) {
        r = a.ranges[row * a.parts + lane];
    }
    const uint64_t* keys = a.keys + row * a.parts * a.top;
    uint64_t part[LOGPROB_PARTS / WAVES];
#pragma unroll
    for (int i = 0; i < LOGPROB_PARTS / WAVES; i++) {
        const uint32_t p = wave + WAVES * i;
        const uint32_t place = i ? 63 - lane : lane;   // the first falling, the others rising
        part[i] = p < a.parts && place < a.top ? keys[(size_t)p * a.top + place] : 0;
    }
    uint64_t key = part[0];
#pragma unroll
    for (int i = 1; i < LOGPROB_PARTS / WAVES; i++) {
        if (wave + WAVES * i < a.parts) {
            key = merge_best(key, part[i], lane);
        }
    }
    if (a.top) {
        key = join_lists(lists, key, a.parts < WAVES ? a.parts : WAVES, wave, lane);
    }
    if (wave) {
        return;
    }
    rescale(r, wave_max64(r.m));
    r.z = wave_sum(r.z);
    r.w = wave_sum(r.w);
    r.bad = __ballot(r.bad != 0) != 0;
    finish(a, row, r, key, lane);
}

}  // namespace lh

using namespace lh;

// Workgroups of a row: one for each unit of the chip in all (256 rows of 131072: 31 us;
// with twice as many 42, a second launch and twice the candidates), each wave with a
// chunk at least.
enum { LOGPROB_WORKGROUPS = 256 };

static uint32_t logprob_parts(uint32_t rows, uint32_t vocab)
{
    const uint32_t chunks = (vocab + CHUNK - 1) / CHUNK, most = (chunks + WAVES - 1) / WAVES;
    uint32_t parts = LOGPROB_WORKGROUPS / rows;
    parts = parts < most ? parts : most;
    parts = parts ? parts : 1;
    return parts < LOGPROB_PARTS ? parts : LOGPROB_PARTS;
}

extern "C" size_t lh_logprobs_scratch_bytes(uint32_t rows, uint32_t vocab, uint32_t top)
{
    const size_t parts = logprob_parts(rows, vocab);
    return parts == 1 ? 0 : lh_round16(rows * parts * (sizeof(Range) + 8 * (size_t)top));
}

extern "C" int lh_launch_logprobs(const float* logits, size_t stride, uint32_t rows,
    uint32_t vocab, const int64_t* tokens, float* logprob, float* entropy, uint32_t top,
    int64_t* top_ids, float* top_logprobs, uint8_t* scratch, hipStream_t s)
{
    const uint32_t parts = logprob_parts(rows, vocab);
    Range* ranges = reinterpret_cast<Range*>(scratch);
    const LogprobArgs a = {logits, tokens, logprob, entropy, top_logprobs, top_ids, ranges,
        reinterpret_cast<uint64_t*>(ranges + (size_t)rows * parts), stride, vocab, top, parts};
    hipLaunchKernelGGL(k_logprob_ranges, dim3(parts, rows), dim3(64 * WAVES), 0, s, a);
    if (const hipError_t e = hipGetLastError()) {
        return (int)e;
    }
    if (parts > 1) {
        hipLaunchKernelGGL(k_logprob_join, dim3(rows), dim3(64 * WAVES), 0, s, a);
    }
    return (int)hipGetLastError();
}
