// Log probabilities, entropy and top alternatives of logit rows (lh_logprobs).
//
// With m = max x and Z = sum e^(x - m): ln p_t = (x_t - m) - ln Z and
// H = ln Z - sum e^(x - m) (x - m) / Z. Both are sums of terms of one sign, so
// nothing cancels; the sums run in 64 bits (as fast as 32 on this chip), which
// keeps ln Z exact where one token has nearly all the probability.
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

// One workgroup a row: the maximum, the sums, then one pass for each place.
__global__ void __launch_bounds__(256)
k_logprobs(const float* __restrict__ logits, size_t stride, uint32_t vocab,
    const int64_t* __restrict__ tokens, float* __restrict__ logprob, float* __restrict__ entropy,
    uint32_t top, int64_t* __restrict__ top_ids, float* __restrict__ top_logprobs)
{
    __shared__ float fmax_[256];
    __shared__ double sums[2][256];
    __shared__ uint64_t keys[256];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const float* x = logits + row * stride;
    float m = -__builtin_inff();
    bool bad = false;
    for (uint32_t i = tid; i < vocab; i += 256) {
        const float v = x[i];
        bad |= !(v < __builtin_inff());
        m = fmaxf(m, v);
    }
    fmax_[tid] = bad ? __builtin_inff() : m;
    __syncthreads();
    for (uint32_t h = 128; h; h >>= 1) {
        if (tid < h) {
            fmax_[tid] = fmaxf(fmax_[tid], fmax_[tid + h]);
        }
        __syncthreads();
    }
    m = fmax_[0];
    bad = m == __builtin_inff();
    const bool empty = m == -__builtin_inff();
    double z = 0, w = 0;
    if (!bad && !empty) {
        for (uint32_t i = tid; i < vocab; i += 256) {
            const float d = x[i] - m, e = expf_cw(d);
            z += e;
            w += e > 0 ? (double)e * d : 0.0;
        }
    }
    sums[0][tid] = z;
    sums[1][tid] = w;
    __syncthreads();
    for (uint32_t h = 128; h; h >>= 1) {
        if (tid < h) {
            sums[0][tid] += sums[0][tid + h];
            sums[1][tid] += sums[1][tid + h];
        }
        __syncthreads();
    }
    const double log_z = log(sums[0][0]);
    const float nan = __builtin_nanf("");
    if (tid == 0 && logprob) {
        const int64_t t = tokens[row];
        float v = nan;
        if (t == -1 && !bad) {
            v = 0;
        } else if (t >= 0 && t < (int64_t)vocab && !bad) {
            v = empty ? -__builtin_inff() : (float)((double)x[t] - m - log_z);
        }
        logprob[row] = v;
    }
    if (tid == 0 && entropy) {
        entropy[row] = bad ? nan : empty ? 0.0f : (float)(log_z - sums[1][0] / sums[0][0]);
    }
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < top; k++) {
        uint64_t best = 0;
        if (!bad && !empty && last) {
            for (uint32_t i = tid; i < vocab; i += 256) {
                const float v = x[i];
                const uint64_t key = v > -__builtin_inff() ? top_key(v, i) : 0;
                best = key < last && key > best ? key : best;
            }
        }
        keys[tid] = best;
        __syncthreads();
        for (uint32_t h = 128; h; h >>= 1) {
            if (tid < h && keys[tid + h] > keys[tid]) {
                keys[tid] = keys[tid + h];
            }
            __syncthreads();
        }
        last = keys[0];
        __syncthreads();
        if (tid == 0) {
            top_ids[(size_t)row * top + k] = last ? (int64_t)(uint32_t)~(uint32_t)last : -1;
            top_logprobs[(size_t)row * top + k] = bad ? nan : !last ? -__builtin_inff()
                : (float)((double)key_logit(last) - m - log_z);
        }
    }
}

}  // namespace lh

using namespace lh;

extern "C" size_t lh_logprobs_scratch_bytes(uint32_t rows, uint32_t vocab, uint32_t top)
{
    (void)rows;
    (void)vocab;
    (void)top;
    return 0;
}

extern "C" int lh_launch_logprobs(const float* logits, size_t stride, uint32_t rows,
    uint32_t vocab, const int64_t* tokens, float* logprob, float* entropy, uint32_t top,
    int64_t* top_ids, float* top_logprobs, uint8_t* scratch, hipStream_t s)
{
    (void)scratch;
    hipLaunchKernelGGL(k_logprobs, dim3(rows), dim3(256), 0, s, logits, stride, vocab, tokens,
        logprob, entropy, top, top_ids, top_logprobs);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
