// Products with 4-bit weights and BF16 group scales (lh_q4_*).
//
// Packed weights: tiles of 16 rows x 128 columns, row tile by row tile, the
// codes of all tiles first. A tile's 1 KiB of codes holds for lane
// l = 16 g + r of a wave 16 bytes: word j has row r's columns 32 j + 8 g .. + 7,
// the even ones' codes in nibbles 0..3 and the odd ones' in 4..7, so that
// (word >> 4 i) & 0x000f000f is columns 2 i and 2 i + 1 as two 16-bit halves: the
// operand of a 16x16x32 matrix instruction. Then the scales: a tile's hold for g
// and group j the four BF16 scales of rows 4 g .. 4 g + 3, the rows of a lane's
// results. Rows and columns past the matrix have code 8 and scale 0.
#include "lh_device.h"
#include "lh_serving.h"

namespace lh {

struct Q4Shape {
    uint32_t rows, cols, group, tiles, blocks;   // 16-row tiles, 128-column blocks
};

static Q4Shape q4_shape(uint32_t rows, uint32_t cols, uint32_t group)
{
    return {rows, cols, group, (rows + 15) / 16, (cols + 127) / 128};
}

__device__ __forceinline__ size_t q4_scales_at(const Q4Shape& p)
{
    return (size_t)p.tiles * p.blocks * 1024;
}

// Byte of (16-row tile, block)'s scale of row r (0..15) and group j of the block.
__device__ __forceinline__ size_t q4_scale_at(const Q4Shape& p, uint32_t tile, uint32_t block,
    uint32_t r, uint32_t j)
{
    const uint32_t per = 128 / p.group;
    return q4_scales_at(p) + ((size_t)tile * p.blocks + block) * (32 * per) +
        ((r >> 2) * per + j) * 8 + (r & 3) * 2;
}

// One word of packed codes a thread: grid (tiles, blocks), 256 threads.
__global__ void __launch_bounds__(256)
k_q4_pack(const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scales, Q4Shape p,
    uint8_t* __restrict__ packed)
{
    const uint32_t tile = blockIdx.x, block = blockIdx.y, i = threadIdx.x;
    const uint32_t lane = i >> 2, j = i & 3, row = tile * 16 + (lane & 15);
    const uint32_t col = block * 128 + 32 * j + 8 * (lane >> 4);
    uint32_t word = 0x88888888u;
    if (row < p.rows && col < p.cols) {
        const uint8_t* c = codes + (size_t)row * (p.cols / 2) + col / 2;
        word = 0;
        for (int e = 0; e < 4; e++) {
            const uint32_t two = c[e];
            word |= (two & 15u) << (4 * e) | (two >> 4) << (16 + 4 * e);
        }
    }
    reinterpret_cast<uint32_t*>(packed)[((size_t)tile * p.blocks + block) * 256 + i] = word;
    const uint32_t per = 128 / p.group;
    if (i < 16 * per) {
        const uint32_t r = i / per, g = i % per, srow = tile * 16 + r, gcol = block * per + g;
        const uint16_t v = srow < p.rows && gcol < p.cols / p.group
            ? scales[(size_t)srow * (p.cols / p.group) + gcol] : (uint16_t)0;
        *reinterpret_cast<uint16_t*>(packed + q4_scale_at(p, tile, block, r, g)) = v;
    }
}

// Rounds FP32 weights: 256 threads of a (block, tile) form the scales of its
// groups, then a packed word each.
__global__ void __launch_bounds__(256)
k_q4_quantize(const float* __restrict__ w, Q4Shape p, uint8_t* __restrict__ packed)
{
    __shared__ float scale[16][4];
    const uint32_t tile = blockIdx.x, block = blockIdx.y, i = threadIdx.x;
    const uint32_t per = 128 / p.group;
    if (i < 16 * per) {
        const uint32_t r = i / per, g = i % per, row = tile * 16 + r;
        const uint32_t first = block * 128 + g * p.group;
        uint32_t s = 0;
        if (row < p.rows && first < p.cols) {
            float most = 0;
            bool finite = true;
            for (uint32_t c = 0; c < p.group; c++) {
                const float v = w[(size_t)row * p.cols + first + c];
                finite &= __builtin_isfinite(v);
                most = fmaxf(most, fabsf(v));
            }
            s = finite ? bf16_nearest(most / 7.0f) : 0x7fc0u;
        }
        scale[r][g] = bf16_to_f32(s);
        *reinterpret_cast<uint16_t*>(packed + q4_scale_at(p, tile, block, r, g)) = (uint16_t)s;
    }
    __syncthreads();
    const uint32_t lane = i >> 2, j = i & 3, row = tile * 16 + (lane & 15);
    const uint32_t col = block * 128 + 32 * j + 8 * (lane >> 4);
    uint32_t word = 0x88888888u;
    if (row < p.rows && col < p.cols) {
        const float s = scale[lane & 15][(32 * j) / p.group];
        if (s > 0) {
            word = 0;
            for (uint32_t e = 0; e < 8; e++) {
                const float v = w[(size_t)row * p.cols + col + e] / s;
                const float code = __builtin_rintf(fminf(fmaxf(v, -7.0f), 7.0f)) + 8.0f;
                word |= (uint32_t)code << (4 * (e >> 1) + 16 * (e & 1));
            }
        }
    }
    reinterpret_cast<uint32_t*>(packed)[((size_t)tile * p.blocks + block) * 256 + i] = word;
}

// One wave a row and token, one packed word a lane at a time.
__global__ void __launch_bounds__(256)
k_q4_rows(const uint8_t* __restrict__ packed, Q4Shape p, const float* __restrict__ x,
    size_t x_stride, float* __restrict__ y, size_t y_stride)
{
    const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const size_t token = blockIdx.y;
    if (row >= p.rows) {
        return;
    }
    const uint32_t tile = row >> 4, r = row & 15;
    float sum = 0;
    for (uint32_t col = lane * 8; col < p.cols; col += 512) {
        const uint32_t block = col >> 7, j = (col >> 5) & 3, g = (col >> 3) & 3;
        const uint32_t word = reinterpret_cast<const uint32_t*>(packed)
            [((size_t)tile * p.blocks + block) * 256 + (g * 16 + r) * 4 + j];
        const float s = bf16_to_f32(*reinterpret_cast<const uint16_t*>(
            packed + q4_scale_at(p, tile, block, r, (col & 127) / p.group)));
        float part = 0;
        for (uint32_t e = 0; e < 8; e++) {
            const int code = (word >> (4 * (e >> 1) + 16 * (e & 1))) & 15;
            const float v = x[token * x_stride + col + e];
            part = __builtin_fmaf((float)(code - 8), v, part);
            part = __builtin_fmaf(0.0f, v, part);   // an Inf is a NaN for the whole row
        }
        sum = __builtin_fmaf(s, part, sum);
    }
    sum = wave_tree64(sum);
    if (lane == 0) {
        y[token * y_stride + row] = sum;
    }
}

}  // namespace lh

using namespace lh;

extern "C" int lh_launch_q4_pack(const uint8_t* codes, const uint16_t* scales, uint32_t rows,
    uint32_t cols, uint32_t group, uint8_t* packed, hipStream_t s)
{
    const Q4Shape p = q4_shape(rows, cols, group);
    hipLaunchKernelGGL(k_q4_pack, dim3(p.tiles, p.blocks), dim3(256), 0, s, codes, scales, p,
        packed);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

extern "C" int lh_launch_q4_quantize(const float* w, uint32_t rows, uint32_t cols, uint32_t group,
    uint8_t* packed, hipStream_t s)
{
    const Q4Shape p = q4_shape(rows, cols, group);
    hipLaunchKernelGGL(k_q4_quantize, dim3(p.tiles, p.blocks), dim3(256), 0, s, w, p, packed);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

extern "C" size_t lh_q4_scratch_bytes(uint32_t cols, uint32_t tokens)
{
    (void)cols;
    (void)tokens;
    return 0;
}

extern "C" int lh_launch_q4_matvec(const uint8_t* packed, const float* x, size_t x_stride,
    float* y, size_t y_stride, uint32_t rows, uint32_t cols, uint32_t group, uint32_t tokens,
    uint8_t* scratch, hipStream_t s)
{
    (void)scratch;
    const Q4Shape p = q4_shape(rows, cols, group);
    hipLaunchKernelGGL(k_q4_rows, dim3((rows + 3) / 4, tokens), dim3(256), 0, s, packed, p, x,
        x_stride, y, y_stride);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
