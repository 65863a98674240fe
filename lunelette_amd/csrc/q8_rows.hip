// Rows of FP32 values rounded to 8-bit codes with a scale each (lh_q8_rows, lh_q8_silu,
// lh_q8_norm).
//
// v = x, SiLU(x) * second, or gamma (h / sqrt(mean h^2 + 1e-5)) with h = x + second;
// scale = max |v| / 127, code = rint(v / scale). A code that lies next to a border
// between two would change with v's last bits, so v is formed in 64 bits, which is as
// fast here as the bytes come.
#include "lh_device.h"
#include "lh_serving.h"

namespace lh {

// Values c .. c + 3 of a row, and whether they are finite.
struct Four {
    double v[4];
    bool finite;
};

template <int KIND>
__device__ __forceinline__ float q8_input(const lh_q8_source& a, size_t row, uint32_t c)
{
    const float x = a.x[row * a.x_stride + c];
    return KIND == LH_Q8_NORM && a.second ? x + a.second[row * a.second_stride + c] : x;
}

// The row's value at c; h of the norm.
template <int KIND>
__device__ __forceinline__ double q8_value(const lh_q8_source& a, size_t row, uint32_t c, float x)
{
    if (KIND == LH_Q8_SILU) {
        return (double)x / (1.0 + exp(-(double)x)) *
            (double)a.second[row * a.second_stride + c];
    }
    return KIND == LH_Q8_NORM ? (double)a.gamma[c] * (double)x : (double)x;
}

// A workgroup a row.
template <int KIND>
__global__ void __launch_bounds__(256)
k_q8_rows(lh_q8_source a)
{
    __shared__ double sums[4], mosts[4];
    __shared__ uint32_t odd;
    const size_t row = blockIdx.x;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) {
        odd = 0;
    }
    __syncthreads();
    double sum = 0, most = 0;
    bool finite = true;
    for (uint32_t c = threadIdx.x; c < a.width; c += 256) {
        const float x = q8_input<KIND>(a, row, c);
        if (KIND == LH_Q8_NORM) {
            if (a.sum) {
                a.sum[row * a.sum_stride + c] = x;
            }
            sum += (double)x * (double)x;
        }
        const double v = q8_value<KIND>(a, row, c, x);
        finite &= __builtin_isfinite(v) && __builtin_isfinite(x);
        most = fmax(most, fabs(v));
    }
    for (int s = 32; s; s >>= 1) {
        sum += __shfl_xor(sum, s);
        most = fmax(most, __shfl_xor(most, s));
    }
    if (lane == 0) {
        sums[wave] = sum;
        mosts[wave] = most;
    }
    if (!finite) {
        odd = 1;
    }
    __syncthreads();
    sum = sums[0] + sums[1] + sums[2] + sums[3];
    most = fmax(fmax(mosts[0], mosts[1]), fmax(mosts[2], mosts[3]));
    const double r = KIND == LH_Q8_NORM ? 1.0 / sqrt(sum / a.width + 1e-5) : 1.0;
    float scale = (float)(most * r / 127.0);
    const bool bad = odd || !__builtin_isfinite(scale);
    if (threadIdx.x == 0) {
        a.scales[row] = bad ? __builtin_nanf("") : scale;
    }
    for (uint32_t c = threadIdx.x; c < a.width; c += 256) {
        double v = 0;
        if (!bad && scale > 0) {
            const float x = KIND == LH_Q8_NORM && a.sum ? a.sum[row * a.sum_stride + c]
                : q8_input<KIND>(a, row, c);
            v = q8_value<KIND>(a, row, c, x) * r / (double)scale;
            v = rint(fmin(fmax(v, -127.0), 127.0));
        }
        a.codes[row * a.code_stride + c] = (int8_t)v;
    }
}

}  // namespace lh

using namespace lh;

extern "C" int lh_launch_q8_rows(int kind, const lh_q8_source* rows, hipStream_t s)
{
    const dim3 grid(rows->tokens), block(256);
    if (kind == LH_Q8_SILU) {
        hipLaunchKernelGGL(k_q8_rows<LH_Q8_SILU>, grid, block, 0, s, *rows);
    } else if (kind == LH_Q8_NORM) {
        hipLaunchKernelGGL(k_q8_rows<LH_Q8_NORM>, grid, block, 0, s, *rows);
    } else {
        hipLaunchKernelGGL(k_q8_rows<LH_Q8_ROWS>, grid, block, 0, s, *rows);
    }
    return (int)hipGetLastError();
}
