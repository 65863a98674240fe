// Log probabilities, entropy and top alternatives of logit rows (lh_logprobs).
//
// With m = max x and Z = sum e^(x - m): ln p_t = (x_t - m) - ln Z and
// H = ln Z - sum e^(x - m) (x - m) / Z. Both are sums of terms of one sign, so
// nothing cancels; the sums run in 64 bits (as fast as 32 on this chip) and the
// largest logit's own term is exactly 1, which keeps ln Z to FP32's relative
// precision where one token has nearly all the probability.
//
// One pass: a row is dealt to workgroups (one or more a row), each wave reads chunks
// of 1024 logits with the running maximum, the two sums and its best `top` keys, and
// they meet in the workgroup and, past one workgroup a row, in a second launch.
#include "lh_device.h"
#include "lh_serving.h"

namespace lh {

// Order of the alternatives as one 64-bit number: the logit's rank (-0 as +0)
// above, the complement of the id below, so a larger key is a likelier token or
// an equal one of lower id. 0 is no token: finite logits have ranks above 0.
__device__ __forceinline__ uint64_t top_key(float v, uint32_t id)
{
    const uint32_t u = __float_as_uint(v + 0.0f);
    const uint32_t rank = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t)rank << 32 | (uint32_t)~id;
}

__device__ __forceinline__ float key_logit(uint64_t key)
{
    const uint32_t rank = (uint32_t)(key >> 32);
    return __uint_as_float(rank & 0x80000000u ? rank & 0x7fffffffu : ~rank);
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

// The 64 lanes' keys in rising order (bitonic network, 21 exchanges).
__device__ __forceinline__ uint64_t sort_rising(uint64_t key, uint32_t lane)
{
    key = half_merge<1>(key, lane, (lane & 2) != 0);
    key = half_merge<2>(key, lane, (lane & 4) != 0);
    key = half_merge<4>(key, lane, (lane & 8) != 0);
    key = half_merge<8>(key, lane, (lane & 16) != 0);
    key = half_merge<16>(key, lane, (lane & 32) != 0);
    return half_merge<32>(key, lane, false);
}

// The best 64 of `best` (falling) and `rising`, falling.
__device__ __forceinline__ uint64_t merge_best(uint64_t best, uint64_t rising, uint32_t lane)
{
    return half_merge<32>(best > rising ? best : rising, lane, true);
}

// Lane l's key of lane 63 - l: a falling list as a rising one.
__device__ __forceinline__ uint64_t reversed(uint64_t key, uint32_t lane)
{
    const int from = (63 - (int)lane) * 4;
    return (uint64_t)(uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(key >> 32)) << 32 |
        (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)key);
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

// Keys that passed a wave's threshold, until 64 of them are sorted into its list.
struct Best {
    volatile uint64_t* buffer;   // 128 of the wave's own
    uint64_t key;                // lane i: the i-th best
    uint64_t least;              // the place `top`, which a key has to pass
    uint32_t count, lane;

    __device__ __forceinline__ void flush(uint32_t top)
    {
        const uint64_t mine = lane < count ? buffer[lane] : 0;
        key = merge_best(key, sort_rising(mine, lane), lane);
        if (count > 64) {
            buffer[lane] = buffer[64 + lane];   // those past the count are never read
            count -= 64;
        } else {
            count = 0;
        }
        const uint64_t last = key;
        least = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(last >> 32), top - 1) << 32 |
            (uint32_t)__builtin_amdgcn_readlane((int)last, top - 1);
    }
    __device__ __forceinline__ void offer(float v, uint32_t id, uint32_t top)
    {
        const uint64_t k = top_key(v, id);
        const bool pass = v > -__builtin_inff() && k > least;
        const uint64_t mask = __ballot(pass);
        if (!mask) {
            return;
        }
        if (pass) {
            buffer[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = k;
        }
        count += __popcll(mask);
        if (count >= 64) {
            flush(top);
        }
    }
};

enum { CHUNK = 1024, WAVES = 4 };

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
            : (float)((double)key_logit(key) - (double)r.m - log_z);
    }
}

// grid (parts, rows), four waves. Whole chunks load 16 bytes a lane, the row's last
// one looks at every id.
__global__ void __launch_bounds__(256)
k_logprob_ranges(LogprobArgs a)
{
    __shared__ uint64_t buffers[WAVES][128];
    __shared__ Range ranges[WAVES];
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const size_t row = blockIdx.y;
    const float* x = a.logits + row * a.stride;
    const uint32_t chunks = (a.vocab + CHUNK - 1) / CHUNK, waves = a.parts * WAVES;
    const uint32_t each = (chunks + waves - 1) / waves;
    uint32_t c = (blockIdx.x * WAVES + wave) * each;
    const uint32_t end = c + each < chunks ? c + each : chunks;
    Range r = {0, 0, -__builtin_inff(), 0};
    Best best = {buffers[wave], 0, 0, 0, lane};
    bool bad = false;
    auto load = [&](uint32_t chunk, float4 (&v)[4]) __attribute__((always_inline)) {
        const uint32_t base = chunk * CHUNK + 4 * lane;
        if ((chunk + 1) * CHUNK <= a.vocab) {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                v[q] = load4(x + base + 256 * q);
            }
        } else {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                float f[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t id = base + 256 * q + i;
                    f[i] = id < a.vocab ? x[id] : -__builtin_inff();
                }
                v[q] = make_float4(f[0], f[1], f[2], f[3]);
            }
        }
    };
    float4 next[4];
    if (c < end) {
        load(c, next);
    }
    for (; c < end; c++) {
        float v[16];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            v[4 * q] = next[q].x, v[4 * q + 1] = next[q].y;
            v[4 * q + 2] = next[q].z, v[4 * q + 3] = next[q].w;
        }
        if (c + 1 < end) {
            load(c + 1, next);
        }
        float most = v[0];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            bad |= !(v[i] < __builtin_inff());
            most = fmaxf(most, v[i]);
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
        if (a.top && __ballot(most >= (best.least ? key_logit(best.least) : -__builtin_inff()))) {
            const uint32_t id = c * CHUNK + 4 * lane;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                best.offer(v[i], id + 256 * (i >> 2) + (i & 3), a.top);
            }
        }
    }
    if (best.count) {
        best.flush(a.top);
    }
    r.bad = __ballot(bad) != 0;
    r.z = wave_sum(r.z);
    r.w = wave_sum(r.w);
    // The waves' lists, falling, in their own buffers.
    best.buffer[lane] = best.key;
    if (lane == 0) {
        ranges[wave] = r;
    }
    __syncthreads();
    if (wave) {
        return;
    }
    float m = r.m;
    uint64_t key = best.key;
    for (int w = 1; w < WAVES; w++) {
        m = fmaxf(m, ranges[w].m);
        if (a.top) {
            key = merge_best(key, buffers[w][63 - lane], lane);
        }
    }
    rescale(r, m);
    for (int w = 1; w < WAVES; w++) {
        Range o = ranges[w];
        rescale(o, m);
        r.z += o.z;
        r.w += o.w;
        r.bad |= o.bad;
    }
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

// Joins a row's parts (at most 64): lane p has part p's range, waves take every fourth
// part's keys.
__global__ void __launch_bounds__(256)
k_logprob_join(LogprobArgs a)
{
    __shared__ uint64_t lists[WAVES][64];
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const size_t row = blockIdx.x;
    uint64_t key = 0;
    if (a.top) {
        const uint64_t* keys = a.keys + row * a.parts * a.top;
        // A list of a part, rising: its place 63 - lane.
        const uint32_t place = 63 - lane;
        uint64_t next = wave < a.parts && place < a.top ? keys[(size_t)wave * a.top + place] : 0;
        for (uint32_t p = wave; p < a.parts; p += WAVES) {
            const uint64_t rising = next;
            const uint32_t after = p + WAVES;
            next = after < a.parts && place < a.top ? keys[(size_t)after * a.top + place] : 0;
            key = merge_best(key, rising, lane);
        }
        lists[wave][lane] = key;
        __syncthreads();
    }
    if (wave) {
        return;
    }
    if (a.top) {
        for (int w = 1; w < WAVES; w++) {
            key = merge_best(key, lists[w][63 - lane], lane);
        }
    }
    Range r = {0, 0, -__builtin_inff(), 0};
    if (lane < a.parts) {
        r = a.ranges[row * a.parts + lane];
    }
    rescale(r, wave_max64(r.m));
    r.z = wave_sum(r.z);
    r.w = wave_sum(r.w);
    r.bad = __ballot(r.bad != 0) != 0;
    finish(a, row, r, key, lane);
}

}  // namespace lh

using namespace lh;

// Workgroups of a row: enough for the whole launch to fill the chip, each wave at
// least one chunk.
enum { LOGPROB_WORKGROUPS = 1024, LOGPROB_PARTS = 64 };

static uint32_t logprob_parts(uint32_t rows, uint32_t vocab)
{
    const uint32_t chunks = (vocab + CHUNK - 1) / CHUNK;
    const uint32_t most = (chunks + WAVES - 1) / WAVES;
    uint32_t parts = (LOGPROB_WORKGROUPS + rows - 1) / rows;
    parts = parts < most ? parts : most;
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
    hipLaunchKernelGGL(k_logprob_ranges, dim3(parts, rows), dim3(256), 0, s, a);
    if (hipGetLastError() != hipSuccess) {
        return -1;
    }
    if (parts > 1) {
        hipLaunchKernelGGL(k_logprob_join, dim3(rows), dim3(256), 0, s, a);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
