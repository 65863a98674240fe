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
// 28.5 us, 4.7 TB/s (27 us without any, 21 us for a plain read of as much); one row is
// two launches and their memory round trips, 11 us.
#include "lh_serving.h"
#include "lh_topk.h"

namespace lh {

enum { LOGPROB_PARTS = 64 };

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
            : (float)((double)rank_logit((uint32_t)(key >> 32)) - (double)r.m - log_z);
    }
}

// grid (parts, rows).
__global__ void __launch_bounds__(64 * WAVES)
k_logprob_ranges(LogprobArgs a)
{
    __shared__ PartShared sh;
    const uint32_t lane = threadIdx.x & 63;
    const size_t row = blockIdx.y;
    Range r;
    uint64_t key;
    scan_part<true>(sh, a.logits + row * a.stride, a.vocab, a.top, blockIdx.x, a.parts, r, key);
    if (threadIdx.x >= 64) {
        return;
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
    r.z = wave_sum(r.z, lane);
    r.w = wave_sum(r.w, lane);
    r.bad = __ballot(r.bad != 0) != 0;
    finish(a, row, r, key, lane);
}

}  // namespace lh

using namespace lh;

// Workgroups of a row: one for each unit of the chip in all (256 rows of 131072: 30 us;
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
